// The states of the gated delta rule, from chunk to chunk, and their gradients the other way
// (include/tops_gla_delta.h; formulas and names in delta_chunk.hip and delta_bwd.hip).
//
// The columns of S and N are independent of one another: a wave owns 16 of them over all
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
//
// A chunk's step of the second pass has, for 128 keys and a wave's 16 values, 188 matrix instructions
// of 16 cycles (states, the system and written values in three parts, what goes into outputs in two), 850
// others, most of them making operands, and 177 LDS accesses. For the two waves of a SIMD these are 6000
// and 6800 cycles, for a CU's LDS 9700, half of them bank conflicts, of the 17500 that a step takes: none of
// the three is full, a wave waits 37 % of its time. Eight waves a block share the tiles, and its halves go
// through the step in different orders, so that one's matrix instructions meet the other's others. 16384
// tokens of 16 heads of 128 x 128: first pass 191 us (29 blocks a head for 16 segments, 464 in two rounds of
// the CUs), second, with the outputs, 151; training of 2 x 4096 tokens: 106 and 110, and the gradients' 70
// and 94. (With every operand in one part less, states 3.5e-6 off and outputs 2.3e-3: 141 and 117.)
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

// Blocks n a segment (or sequence): its neighbouring heads and columns, which read the same keys, go
// to one XCD, and every XCD has a part of every segment. (Whole segments to an XCD: a sequence of
// 200 chunks behind 40 of 4 had one XCD at work, 1083 us a call, so 393; equal ones the same.)
__device__ __forceinline__ int spread(int blk, int n) {
  const int r = blk % n;
  return blk - r + xcd_remap(r, n);
}

// Where a map's element (row, col) lies: in the order of the fold's operands (rows of pair_row, 8
// columns a lane), so that a wave's load is 1024 bytes side by side.
template <int KP>
__device__ __forceinline__ int map_at(int row, int col) {
  const int lane = 16 * (col >> 3 & 3) + 4 * (row >> 3 & 3) + (row & 3);
  return (((row >> 5) * 2 + (row >> 2 & 1)) * (KP / 32) + (col >> 5)) * 512 + 8 * lane + (col & 7);
}

// A head's columns go to blocks of NW waves of 16, of V or, in a first pass, then of KP for M.
template <typename T, int KP, int NW>
struct ScanShape {
  static constexpr int C = delta_c<T>(), COLS = 16 * NW;
  static constexpr int PK = pitch_of<T>(KP), PT = pitch_of<T>(32), PV = pitch_of<T>(COLS);
  static constexpr int NT = 64 * NW, TRI = delta_blocks<T>() * 32;   // rows of a part of Tm or P
  static constexpr int PART = TRI * PT;   // from a part to the next one
};
constexpr int LDS_MOST = 160 * 1024;

template <typename T>
__device__ __forceinline__ T* at_off(char* base, uint32_t off) {
  return (T*)(base + off);
}
// The first n of 8 elements to any address of theirs.
template <typename T>
__device__ __forceinline__ void put_frag(T* p, const Frag<T>& f, int n) {
  const Run<T, 8> r = __builtin_bit_cast(Eight<T>, f);
  if (n >= 8) {
    *reinterpret_cast<Run<T, 8>*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = r.v[e];
  }
}

// FIRST: the first pass, which has E (and M) and no outputs.
template <typename T, int KP, int NW, bool FIRST>
struct ScanLds : ScanShape<T, KP, NW> {
  using B = ScanShape<T, KP, NW>;
  static constexpr int C = B::C, ES = (int)sizeof(T);
  static constexpr int K0 = 0, T0 = C * B::PK, V0 = T0 + WHOLE<T> * B::PART, END = V0 + C * B::PV;
  static constexpr int F0 = END * ES;   // five vectors of floats
  static constexpr int ONE = F0 + 5 * C * 4;
  // the scores' part: q, two parts of P, the sums of log decays, 1 / |q|
  static constexpr int Q0 = 0, P0 = C * B::PK, G0 = (P0 + TWO<T> * B::PART) * ES, R0 = G0 + 8 * C;
  static constexpr int REST = FIRST ? 0 : R0 + 4 * C;
  static constexpr int BUFS = 2 * ONE + REST + (2 + B::COLS) * 4 <= LDS_MOST ? 2 : 1;   // of the chunk's tiles
  static constexpr int BYTES = BUFS * ONE + REST + (2 + B::COLS) * 4;
  static_assert(BYTES <= LDS_MOST && ONE % 16 == 0 && G0 % 8 == 0, "LDS");
};

template <typename T, int KP, int NW, bool FIRST>
__global__ __launch_bounds__(64 * NW) void delta_scan_kernel(DeltaParams p) {
  using L = ScanLds<T, KP, NW, FIRST>;
  constexpr int C = L::C, NT = L::NT, NS = KP / 32, NU = C / 32, COLS = L::COLS, ES = L::ES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, ci = lane & 15;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + COLS - 1) / COLS, mt = FIRST ? (KP + COLS - 1) / COLS : 0;
  int blk = spread((int)blockIdx.x, (vt + mt) * HV);
  const int vb = blk % (vt + mt);
  blk /= vt + mt;
  const int hv = blk % HV, h = hv / (HV / (int)a.H);
  const SegAt at = seg_at(a, C, blk / HV);
  const bool map = FIRST && vb >= vt;   // columns of M
  if (FIRST && (at.j + 1 >= at.count || (map && at.j == 0))) return;   // nobody asks for these
  const int nc = at.n;
  const T* kp = (const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh;
  const T* qp = (const T*)a.q + at.b * a.q_sb + at.t * a.q_st + h * a.q_sh;
  // the block's columns; the last block's few may begin before them, where there are fewer than 8
  const int vc = map ? COLS : V - vb * COLS;
  const T* vp = (const T*)a.v + at.b * a.v_sb + at.t * a.v_st + hv * a.v_sh + (map ? 0 : vb * COLS);
  const int w0 = 16 * wave, v = (map ? vb - vt : vb) * COLS + w0 + ci;
  const bool idle = v - ci >= (map ? KP : V);   // a wave past the columns only helps with the tiles
  const bool vin = v < V;

  f32x4 S[2 * NS];
  const float* from = nullptr;
  if (at.j > 0) {
    if (!FIRST) from = p.E + ((long)(at.seg - 1) * HV + hv) * K * V;
  } else if (a.h0) {
    from = a.h0 + ((long)at.seq * HV + hv) * K * V;
  }
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[i][r] = map && v == 32 * (i >> 1) + 8 * g + 4 * (i & 1) + r ? 1.f : 0.f;
  if (from && !map) load_state(S, from + min(v, V - 1), vin, g, K, V);

  // byte offsets of a lane's stores from bases that are the same for all
  const uint32_t s_off = (uint32_t)(v * TWO<T> * KP + 8 * g) * ES;
  const uint32_t n_off = (uint32_t)(v * TWO<T> * C + 8 * g) * ES;
  const uint32_t o_off =
      (uint32_t)(tid / (COLS / 8) * HV * V + vb * COLS + tid % (COLS / 8) * 8) * ES;
  TileStream<T, C, KP, NT> fk(a.k_st, K, tid), fq(a.q_st, K, tid);
  BlockStream<T, WHOLE<T> * L::TRI, NT> ft;
  TileStream<T, C, COLS, NT> fv(a.v_st, vc, tid);
  constexpr int NF = (5 * C + NT - 1) / NT;
  float ff[NF];
  double fg = 0.;
  int fin = 0;   // tokens before the first one that is not finite
  // where the next chunk's inputs lie, and this chunk's other parts; all of them go on by their steps
  const long unit0 = (long)at.chunk * HV + hv;
  const int k_st = (int)a.k_st, q_st = (int)a.q_st, v_st = (int)a.v_st;
  const char* Tn = p.Tm + unit0 * p.tri_bytes;
  const char* vecn = p.vec + unit0 * p.vec_bytes;
  char *vecc = p.vec + unit0 * p.vec_bytes, *Pc = p.P + unit0 * p.tri_bytes;
  char *Sc = p.S + unit0 * V * KP * TWO<T> * ES, *Nc = p.N + unit0 * V * C * TWO<T> * ES;
  char* oc = (char*)a.o + (((long)at.b * a.T + at.t) * HV + hv) * V * ES;
  const long t_step = (long)HV * p.tri_bytes, vec_step = (long)HV * p.vec_bytes;
  const long s_step = (long)HV * V * KP * TWO<T> * ES, n_step = (long)HV * V * C * TWO<T> * ES;
  const int o_row = HV * V * ES;   // and a row of o
  const float scale = (float)a.scale;
  const bool l2norm = a.l2norm != 0, keep = a.train != 0, keep_p = keep && vb == 0;
  // in two lots in the second pass, as the loads of all waves at once hold up the waves
  auto fetch = [&](int len) {
    fk.next(kp, k_st, len);
    kp += (long)C * k_st;
    if (!map) {
      fv.next(vp, v_st, len);
      vp += (long)C * v_st;
    }
  };
  auto fetch2 = [&](int len) {
    ft.next((const T*)Tn, tid);
    const float* vec = (const float*)vecn;
#pragma unroll
    for (int i = 0; i < NF; ++i) ff[i] = vec[min(i * NT + tid, 5 * C - 1)];
    fin = *(const int*)(vecn + 36 * C);
    if (!FIRST) {
      fq.next(qp, q_st, len);
      qp += (long)C * q_st;
      fg = ((const double*)(vecn + 28 * C))[min(tid, C - 1)];
    }
    Tn += t_step;
    vecn += vec_step;
  };
  unsigned char* rest = smem + L::BUFS * L::ONE;
  T *sQ = (T*)rest + L::Q0, *sP = (T*)rest + L::P0;
  double* sG = (double*)(rest + L::G0);
  float* sRq = (float*)(rest + L::R0);
  // chunks with values that are not finite, by turns, and from which token on each column has them
  int *sFlag = (int*)(smem + L::BYTES - (2 + COLS) * 4), *sFirst = sFlag + 2;
  auto put = [&](unsigned char* buf, int len, int n) {
    T* sm = (T*)buf;
    const int rows = min(len, __builtin_amdgcn_readfirstlane(fin));
    fk.put(sm + L::K0, L::PK, rows, K, tid);
    ft.put(sm + L::T0, L::PT, tid);
    fv.put(sm + L::V0, L::PV, map ? 0 : rows, vc, tid);
    if (!map && fv.not_finite()) sFlag[n & 1] = n;
    float* sf = (float*)(buf + L::F0);
#pragma unroll
    for (int i = 0; i < NF; ++i)
      if (i * NT + tid < 5 * C) sf[i * NT + tid] = ff[i];
    if (!FIRST) {
      fq.put(sQ, L::PK, len, K, tid);
      if (tid < C) sG[tid] = fg;
    }
  };
  // a chunk's outputs, which its waves left where its values were, in whole rows
  auto store_o = [&](const unsigned char* buf, int len) {
    constexpr int ROWS = NT / (COLS / 8);
    const int row = tid / (COLS / 8), col = tid % (COLS / 8) * 8;
    const T* so = (const T*)buf + L::V0 + row * L::PV + col;
    if (col < vc) {
#pragma unroll
      for (int i = 0; i < C / ROWS; ++i)
        if (row + i * ROWS < len)
          put_frag(at_off<T>(oc + (long)(i * ROWS) * o_row, o_off),
                   ld_frag(so + i * ROWS * L::PV), vc - col);
    }
    oc += (long)C * o_row;
  };
  // The scores of 16 tokens (columns) with 32 before or among them (rows), of six such items in a
  // chunk of 64 and two in one of 32: a lane has 8 in a row of P.
  auto scores = [&](int it, const T* sK, const float* sf) {
    const int u = it >= 4, tile = it < 4 ? it : it - 2, i = 16 * tile + ci, j0 = 32 * u + 8 * g;
    f32x4 acc[2] = {zero4(), zero4()};
    float qq = 0.f;
#pragma unroll
    for (int s0 = 0; s0 < NS; s0 += 4) {
      constexpr int B = NS < 4 ? NS : 4;   // a few reads on their way at once
      Frag<T> qf[B], kf[B][2];
#pragma unroll
      for (int s = 0; s < B; ++s) {
        qf[s] = ld_frag(sQ + i * L::PK + 32 * (s0 + s) + 8 * g);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          kf[s][x] = ld_frag(sK + (32 * u + pair_row(lane, x)) * L::PK + 32 * (s0 + s) + 8 * g);
      }
#pragma unroll
      for (int s = 0; s < B; ++s) {
        mma(acc[0], kf[s][0], qf[s]);
        mma(acc[1], kf[s][1], qf[s]);
      }
#pragma unroll
      for (int s = 0; s < B; ++s) {
        float x[8];
        values_of(qf[s], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) qq = fmaf(x[e], x[e], qq);
      }
    }
    qq = swap32_add(qq, qq);
    qq = swap16_add(qq, qq);
    const float rq = l2norm ? rsqrtf(qq + DELTA_L2_EPS) : 1.f, fq = scale * rq;
    if (u == 0 && g == 0) {
      sRq[i] = fq * sf[4 * C + i];
      if (keep_p) ((float*)vecc)[6 * C + i] = rq;
    }
    float x[8], d[8], rk[8];
    decays<T>(sG[i], sG + j0, 1.f, d);
    ld_eight(sf + 3 * C + j0, rk);
    pair_values(acc[0], acc[1], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = j0 + e <= i ? x[e] * (fq * rk[e] * d[e]) : 0.f;
    const Whole<T> f = split_of<T, WHOLE<T>>(x);
    const int row = 32 * tri_block(tile / 2, u) + i % 32;
#pragma unroll
    for (int part = 0; part < TWO<T>; ++part)
      st_frag(sP + part * L::PART + row * L::PT + 8 * g, f.p[part]);
    if (keep_p) {
      T* out = at_off<T>(Pc, (uint32_t)(row * 32 + 8 * g) * ES);
#pragma unroll
      for (int part = 0; part < WHOLE<T>; ++part) st_frag(out + part * L::TRI * 32, f.p[part]);
    }
  };
  unsigned char *buf = smem, *other = smem + (L::BUFS - 1) * L::ONE;   // this chunk's, the next one's
  int left = at.T;   // tokens from this chunk on
  if (nc > 0) {
    fetch(left);
    fetch2(left);
    if (tid < 2) sFlag[tid] = -1;
    __syncthreads();
    put(buf, left, 0);
  }
  for (int n = 0; n < nc; ++n, left -= C) {
    const bool more = n + 1 < nc;
    __syncthreads();
    // Products would take a value that is not finite to all tokens of its column, so it and what
    // follows it there are left out, and what is made of them is set to NaN.
    const bool spoilt = __builtin_amdgcn_readfirstlane(sFlag[n & 1]) == n;
    if (__builtin_expect(spoilt && !idle, 0)) {
      T* at0 = (T*)buf + L::V0 + w0 + ci;
      int first = C;
#pragma unroll 1
      for (int t = C - 4 + g; t >= 0; t -= 4)
        if (!(fabsf(to_f32(at0[t * L::PV])) < INFINITY)) first = t;
      first = min(first, __shfl_xor(first, 16));
      first = min(first, __shfl_xor(first, 32));
#pragma unroll 1
      for (int t = first; t < C; ++t) at0[t * L::PV] = zero_elem<T>();
      sFirst[w0 + ci] = first;
    }
    // The two halves of the block's waves, one of each on a SIMD, go through a chunk in different
    // orders, so that loads, products and conversions of one lie beside others of the other.
    const bool early = wave < NW / 2;
    auto aside = [&]() {
      if (more) fetch(left - C);
      if (FIRST && more) fetch2(left - C);
      if constexpr (!FIRST) {
        constexpr int ITEMS = NU == 2 ? 6 : 2;
        if (L::BUFS == 2 && n > 0) store_o(other, C);
        if (ITEMS % NW == 0 || wave < ITEMS) scores(wave, (const T*)buf + L::K0, (const float*)(buf + L::F0));
        if (ITEMS > NW && wave + NW < ITEMS) scores(wave + NW, (const T*)buf + L::K0, (const float*)(buf + L::F0));
      }
    };
    if (early) aside();
    const T *sm = (const T*)buf, *sK = sm + L::K0, *sT = sm + L::T0, *sV = sm + L::V0 + w0;
    const float* sf = (const float*)(buf + L::F0);   // e^G / |k|, e^{G_C - G} / |k|, beta, 1 / |k|,
    const float last = sf[5 * C - 1];                // e^G
    f32x4 acc[2 * NU], o[FIRST ? 1 : 2 * NU];
    Two<T> nf[NU];
    if (idle && !early) aside();
    if (!idle) {
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i) acc[i] = o[FIRST ? 0 : i] = zero4();
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        float x[8];
        pair_values(S[2 * s], S[2 * s + 1], x);
        const Whole<T> f = split_of<T, WHOLE<T>>(x);
        mma_rows(acc, [&](int i) {
          return ld_frag(sK + (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PK + 32 * s + 8 * g);
        }, f);
        if constexpr (!FIRST) {
          if (keep && vin)
#pragma unroll
            for (int part = 0; part < TWO<T>; ++part)
              st_frag(at_off<T>(Sc, s_off) + part * KP + 32 * s, f.p[part]);
          mma_rows(o, [&](int i) {
            return ld_frag(sQ + (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PK + 32 * s + 8 * g);
          }, two_of<T>(f));
        }
      }
      if (!early) aside();
      if (!FIRST && more) fetch2(left - C);
      Whole<T> R[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        float x[8], y[8];
        values_of(ld_frag_t(sV + 32 * u * L::PV, L::PV, lane), y);
        pair_values(acc[2 * u], acc[2 * u + 1], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = 32 * u + 8 * g + e;
          x[e] = sf[2 * C + t] * (y[e] - sf[t] * x[e]);
        }
        R[u] = split_of<T, WHOLE<T>>(x);
      }
#pragma unroll
      for (int i = 0; i < 2 * NU; ++i) acc[i] = zero4();
#pragma unroll
      for (int w = 0; w < NU; ++w)
#pragma unroll
        for (int u = w; u < NU; ++u)
          mma_split_pair(acc, u, [&](int x) {
            return ld_split<T, WHOLE<T>>(sT, L::PART,
                                         (32 * tri_block(u, w) + pair_row(lane, x)) * L::PT + 8 * g);
          }, R[w]);
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) S[i] *= last;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        float x[8];
        pair_values(acc[2 * u], acc[2 * u + 1], x);
        if constexpr (!FIRST) {
          nf[u] = split_of<T, TWO<T>>(x);
          if (keep && vin)
#pragma unroll
            for (int part = 0; part < TWO<T>; ++part)
              st_frag(at_off<T>(Nc, n_off) + part * C + 32 * u, nf[u].p[part]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= sf[C + 32 * u + 8 * g + e];
        mma_rows(S, [&](int i) {
          return ld_pair_t(sK + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
        }, split_of<T, WHOLE<T>>(x));
      }
      if (__builtin_expect(spoilt, 0)) {
        const int first = sFirst[w0 + ci];
        if (!FIRST && keep && vin)
#pragma unroll 1
          for (int i = 0; i < 8 * NU; ++i) {   // the tokens that the lane has stored
            const int t = 32 * (i >> 3) + 8 * g + (i & 7);
            if (t >= first) at_off<T>(Nc, n_off)[t - 8 * g] = from_f32<T>(NAN);
          }
        const float x = first < C ? NAN : 1.f;
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) S[i] *= x;
      }
    }
    if constexpr (!FIRST) {
      __syncthreads();   // the scores are there, and no values are read any more
      if (!idle) {
        T* so = (T*)buf + L::V0 + w0 + ci;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          float f[8];
          ld_eight(sRq + 32 * u + 8 * g, f);
#pragma unroll
          for (int x = 0; x < 8; ++x) o[2 * u + x / 4][x % 4] *= f[x];
        }
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int w = 0; w <= u; ++w)
            mma_split_pair(o, u, [&](int x) {
              return ld_split<T, TWO<T>>(sP, L::PART,
                                         (32 * tri_block(u, w) + pair_row(lane, x)) * L::PT + 8 * g);
            }, nf[w]);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int x = 0; x < 8; ++x)
            so[(32 * u + 8 * g + x) * L::PV] = from_f32<T>(o[2 * u + x / 4][x % 4]);
        if (__builtin_expect(spoilt, 0))
#pragma unroll 1
          for (int i = 0; i < 8 * NU; ++i) {
            const int t = 32 * (i >> 3) + 8 * g + (i & 7);
            if (t >= sFirst[w0 + ci]) so[t * L::PV] = from_f32<T>(NAN);
          }
      }
    }
    if (more) {
      if (!FIRST && idle) fetch2(left - C);
      // the scores' tiles have been read (their barrier is behind, or there is none of them); with
      // one buffer, so must the chunk's be, and its outputs
      if (L::BUFS == 1) {
        __syncthreads();
        if (!FIRST) {
          store_o(buf, C);
          __syncthreads();
        }
      }
      put(other, left - C, n + 1);
      unsigned char* x = buf;
      buf = other;
      other = x;
    }
    vecc += vec_step;
    Pc += t_step;
    Sc += s_step;
    Nc += n_step;
  }
  if (!FIRST && nc > 0) {
    __syncthreads();
    store_o(buf, left + C);
  }
  if (idle) return;
  if (map) {   // column v, rows in the lane's order
    constexpr int TILE = KP * KP;
    T* M = (T*)(p.M + ((long)at.seg * HV + hv) * p.map_bytes);
    T* Mt = (T*)(p.Mt + ((long)at.seg * HV + hv) * p.map_bytes);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float x[8], y[8];
      pair_values(S[2 * s], S[2 * s + 1], x);
      const Whole<T> f = split_of<T, WHOLE<T>>(x);
      const int row = 32 * s + 8 * g;
#pragma unroll
      for (int part = 0; part < WHOLE<T>; ++part) {
        if (a.train) st_frag(Mt + part * TILE + map_at<KP>(v, row), f.p[part]);
        values_of(f.p[part], y);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          M[part * TILE + map_at<KP>(row + e, v)] = from_f32<T>(y[e]);
      }
    }
  } else if (FIRST) {
    store_state(S, p.E + ((long)at.seg * HV + hv) * K * V + v, vin, g, K, V);
  } else if (a.ht && at.j + 1 == at.count) {
    store_state(S, a.ht + ((long)at.seq * HV + hv) * K * V + v, vin, g, K, V);
  }
}

template <typename T, int KP, int NW>
struct DscanLds : ScanShape<T, KP, NW> {
  using B = ScanShape<T, KP, NW>;
  static constexpr int C = B::C;
  static constexpr int K0 = 0, Q0 = C * B::PK, T0 = 2 * C * B::PK, P0 = T0 + WHOLE<T> * B::PART;
  static constexpr int V0 = P0 + WHOLE<T> * B::PART, END = V0 + C * B::PV;
  static constexpr int F0 = END * (int)sizeof(T);   // three vectors of floats, e^{G_C}
  static constexpr int BYTES = F0 + (3 * C + 1) * 4;
  static_assert(BYTES <= LDS_MOST, "LDS");
};

template <typename T, int KP, int NW, bool FIRST>
__global__ __launch_bounds__(64 * NW) void delta_dscan_kernel(DeltaParams p) {
  using L = DscanLds<T, KP, NW>;
  constexpr int C = L::C, NT = L::NT, NS = KP / 32, NU = C / 32, COLS = L::COLS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, ci = lane & 15;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + COLS - 1) / COLS;
  int blk = spread((int)blockIdx.x, vt * HV);
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
  const int w0 = 16 * wave, v = vb * COLS + w0 + ci;
  const bool idle = v - ci >= V, vin = v < V;

  f32x4 S[2 * NS];   // dS, as the forward's states
  const float* from = nullptr;
  if (at.j + 1 < at.count) {
    if (!FIRST) from = p.dE + ((long)(at.seg + 1) * HV + hv) * K * V;
  } else if (a.dht) {
    from = a.dht + ((long)at.seq * HV + hv) * K * V;
  }
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i) S[i] = zero4();
  if (from) load_state(S, from + min(v, V - 1), vin, g, K, V);

  TileStream<T, C, KP, NT> fk(a.k_st, K, tid), fq(a.q_st, K, tid);
  BlockStream<T, WHOLE<T> * L::TRI, NT> ft, fp;
  TileStream<T, C, COLS, NT> fd(a.do_st, vc, tid);
  constexpr int ES = (int)sizeof(T);
  const uint32_t s_off = (uint32_t)(v * TWO<T> * KP + 8 * g) * ES;
  const uint32_t n_off = (uint32_t)(v * TWO<T> * C + 8 * g) * ES;
  // where the chunk before has its inputs, and this chunk its outputs; all go back by their steps
  const long unit0 = (long)(at.chunk + nc - 1) * HV + hv;
  const int k_st = (int)a.k_st, q_st = (int)a.q_st, d_st = (int)a.do_st;
  kp += (long)(nc - 1) * C * k_st;
  qp += (long)(nc - 1) * C * q_st;
  dp += (long)(nc - 1) * C * d_st;
  const char *Tn = p.Tm + unit0 * p.tri_bytes, *Pn = p.P + unit0 * p.tri_bytes;
  const char* vecn = p.vec + unit0 * p.vec_bytes;
  char *Sc = p.dS + unit0 * V * KP * TWO<T> * ES, *Yc = p.Y + unit0 * V * C * TWO<T> * ES;
  const long t_step = (long)HV * p.tri_bytes, vec_step = (long)HV * p.vec_bytes;
  const long s_step = (long)HV * V * KP * TWO<T> * ES, n_step = (long)HV * V * C * TWO<T> * ES;
  const float scale = (float)a.scale;
  constexpr int NF = (3 * C + NT) / NT;
  float ff[NF], fr[NF];
  auto fetch = [&](int len) {
    fk.next(kp, k_st, len);
    fd.next(dp, d_st, len);
    kp -= (long)C * k_st;
    dp -= (long)C * d_st;
  };
  auto fetch2 = [&](int len) {
    fq.next(qp, q_st, len);
    ft.next((const T*)Tn, tid);
    fp.next((const T*)Pn, tid);
    const float* vec = (const float*)vecn;
#pragma unroll
    for (int i = 0; i < NF; ++i) {   // e^{G_C - G} / |k|, beta e^G / |k|, scale e^G / |q|; e^{G_C}
      const int x = i * NT + tid, t = x % C;
      ff[i] = vec[x < C ? C + t : x < 2 * C ? t : x < 3 * C ? 4 * C + t : 5 * C - 1];
      fr[i] = vec[x < 2 * C ? 2 * C + t : 6 * C + t];
    }
    qp -= (long)C * q_st;
    Tn -= t_step;
    Pn -= t_step;
    vecn -= vec_step;
  };
  T* sm = (T*)smem;
  T *sK = sm + L::K0, *sQ = sm + L::Q0, *sT = sm + L::T0, *sP = sm + L::P0, *sV = sm + L::V0;
  float* sf = (float*)(smem + L::F0);
  int len = at.T - (nc - 1) * C;   // of the last chunk alone less than C
  if (nc > 0) {
    fetch(len);
    fetch2(len);
  }
  for (int n = nc - 1; n >= 0; --n, len = C) {
    __syncthreads();
    fk.put(sK, L::PK, len, K, tid);
    fq.put(sQ, L::PK, len, K, tid);
    ft.put(sT, L::PT, tid);
    fp.put(sP, L::PT, tid);
    fd.put(sV, L::PV, len, vc, tid);
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const int x = i * NT + tid;
      if (x <= 3 * C)
        sf[x] = x < C || x == 3 * C ? ff[i] : ff[i] * fr[i] * (x < 2 * C ? 1.f : scale);
    }
    __syncthreads();
    if (n > 0) fetch(C);
    if (idle) {
      if (n > 0) fetch2(C);
      continue;
    }
    const float last = sf[3 * C];

    f32x4 acc[2 * NU];
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i) acc[i] = zero4();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float x[8];
      pair_values(S[2 * s], S[2 * s + 1], x);
      const Whole<T> f = split_of<T, WHOLE<T>>(x);
      if (!FIRST && vin)
#pragma unroll
        for (int part = 0; part < TWO<T>; ++part)
          st_frag(at_off<T>(Sc, s_off) + part * KP + 32 * s, f.p[part]);
      mma_rows(acc, [&](int i) {
        return ld_frag(sK + (32 * (i >> 1) + pair_row(lane, i & 1)) * L::PK + 32 * s + 8 * g);
      }, f);
    }
    Frag<T> df[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) df[u] = ld_frag_t(sV + w0 + 32 * u * L::PV, L::PV, lane);
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][r] *= sf[32 * (i >> 1) + 8 * g + 4 * (i & 1) + r];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int w = 0; w <= u; ++w)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          mma(acc[2 * w + x],
              ld_split_t<T, WHOLE<T>>(sP + 32 * tri_block(u, w) * L::PT, L::PART, L::PT, lane, x),
              df[u]);
    if (n > 0) fetch2(C);
    Whole<T> R[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float x[8];
      pair_values(acc[2 * u], acc[2 * u + 1], x);
      R[u] = split_of<T, WHOLE<T>>(x);
    }
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i) acc[i] = zero4();
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int w = 0; w <= u; ++w)
        mma_split_pair(acc, w, [&](int x) {
          return ld_split_t<T, WHOLE<T>>(sT + 32 * tri_block(u, w) * L::PT, L::PART, L::PT, lane, x);
        }, R[u]);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) S[i] *= last;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float x[8];
      values_of(df[u], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= sf[2 * C + 32 * u + 8 * g + e];
      mma_rows(S, [&](int i) {
        return ld_pair_t(sQ + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
      }, split_of<T, WHOLE<T>>(x));
      pair_values(acc[2 * u], acc[2 * u + 1], x);
      if (!FIRST && vin) {
        const Two<T> y = split_of<T, TWO<T>>(x);
#pragma unroll
        for (int part = 0; part < TWO<T>; ++part)
          st_frag(at_off<T>(Yc, n_off) + part * C + 32 * u, y.p[part]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= -sf[C + 32 * u + 8 * g + e];
      mma_rows(S, [&](int i) {
        return ld_pair_t(sK + 32 * u * L::PK + 32 * (i >> 1), L::PK, lane, i & 1);
      }, split_of<T, WHOLE<T>>(x));
    }
    Sc -= s_step;
    Yc -= n_step;
  }
  if (idle) return;
  float* to = FIRST ? p.dE + ((long)at.seg * HV + hv) * K * V
              : a.dh0 && at.j == 0 ? a.dh0 + ((long)at.seq * HV + hv) * K * V : nullptr;
  if (to) store_state(S, to + v, vin, g, K, V);
}

// E_j <- M_j E_{j-1} + E_j along the segments of a sequence and head, or dE_j <- M_j^T dE_{j+1} +
// dE_j the other way. A block has 16 columns, each of its waves 32 of the rows; the
// states go from wave to wave through LDS as operands, the maps and parts of the next segment are
// on their way meanwhile. Bound by the maps' way through the caches, each read by every block of the
// head: 16 segments of 16 heads of 128 x 128 in 31 us (with maps in two parts 22, in rows, 64 bytes a
// row and load, 33; two segments ahead so 40).
template <typename T, int KP, bool BACK>
__global__ __launch_bounds__(delta_fold_threads(KP)) void delta_fold_kernel(DeltaParams p) {
  constexpr int NS = KP / 32, PARTS = WHOLE<T>;
  __shared__ __attribute__((aligned(16))) Frag<T> sh[2][PARTS][NS][64];
  const tops_gla_delta_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int K = (int)a.K, V = (int)a.V, HV = (int)a.HV;
  const int vt = (V + 15) / 16;
  int blk = spread((int)blockIdx.x, vt * HV);
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
  const int k0 = wave * 32;   // the wave's rows: k0 + 8 g + 4 h + r as ever
  auto state = [&](int n) {
    const int j = BACK ? count - 1 - n : n;
    return (BACK ? p.dE : p.E) + ((long)(first + j) * HV + hv) * K * V;
  };
  Whole<T> M[2][NS];
  f32x4 E[2];
  auto fetch = [&](int n) {
    const int j = BACK ? count - 1 - n : n;
    const T* m = (const T*)((BACK ? p.Mt : p.M) + ((long)(first + j) * HV + hv) * p.map_bytes);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s)
        M[i][s] = ld_split<T, PARTS>(m, KP * KP, ((wave * 2 + i) * NS + s) * 512 + 8 * lane);
    load_rows(E, state(n) + min(v, V - 1), k0 + 8 * g, K, V);
  };
  auto share = [&](int n) {   // the wave's rows of the state after step n, and to memory
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = v < V && k0 + 8 * g + e < K ? E[e / 4][e % 4] : 0.f;
    const Whole<T> f = split_of<T, PARTS>(x);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) sh[n & 1][part][wave][lane] = f.p[part];
    if (n > 0 && v < V) store_rows(E, state(n) + v, k0 + 8 * g, K, V);
  };
  load_rows(E, state(0) + min(v, V - 1), k0 + 8 * g, K, V);
  share(0);
  fetch(1);
  for (int n = 1; n + 1 < count; ++n) {
    __syncthreads();
    f32x4 acc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[i] = E[i];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      Whole<T> f;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) f.p[part] = sh[(n - 1) & 1][part][s][lane];
#pragma unroll
      for (int i = 0; i < 2; ++i) mma(acc[i], M[i][s], f);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) E[i] = acc[i];
    share(n);
    if (n + 2 < count) fetch(n + 1);
  }
}

template <typename T, int KP, int NW, bool BACK, bool FIRST>
hipError_t launch(const DeltaParams& p, hipStream_t st) {
  using S = ScanShape<T, KP, NW>;
  constexpr int lds = BACK ? (int)DscanLds<T, KP, NW>::BYTES : (int)ScanLds<T, KP, NW, FIRST>::BYTES;
  const void* f;
  if constexpr (BACK)
    f = (const void*)delta_dscan_kernel<T, KP, NW, FIRST>;
  else
    f = (const void*)delta_scan_kernel<T, KP, NW, FIRST>;
  const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const long cols = (p.a.V + S::COLS - 1) / S::COLS +
                    (FIRST && !BACK ? (KP + S::COLS - 1) / S::COLS : 0);
  const unsigned grid = (unsigned)(cols * p.a.HV * p.a.nsegs);
  if constexpr (BACK)
    delta_dscan_kernel<T, KP, NW, FIRST><<<grid, S::NT, lds, st>>>(p);
  else
    delta_scan_kernel<T, KP, NW, FIRST><<<grid, S::NT, lds, st>>>(p);
  return hipGetLastError();
}

template <typename T, int KP, int NW, bool BACK>
hipError_t passes(const DeltaParams& p, hipStream_t st) {
  if (p.multi) {
    if (const hipError_t e = launch<T, KP, NW, BACK, true>(p, st)) return e;
    const unsigned grid = (unsigned)((p.a.V + 15) / 16 * p.a.HV * p.a.nseq);
    delta_fold_kernel<T, KP, BACK><<<grid, delta_fold_threads(KP), 0, st>>>(p);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return launch<T, KP, NW, BACK, false>(p, st);
}

template <typename T, int KP, bool BACK>
hipError_t run(const DeltaParams& p, hipStream_t st) {
  // eight waves a block share the chunk's tiles, two waves a SIMD; with 256 keys a wave's state
  // leaves no room for a second one
  if constexpr (KP < 256)
    if (p.a.V > 64) return passes<T, KP, 8, BACK>(p, st);
  return passes<T, KP, 4, BACK>(p, st);
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
