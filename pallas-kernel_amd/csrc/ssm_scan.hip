// Selective state space scan, forward and backward (include/tops_gla_ssm.h has the formulas).
//
// A lane owns one channel and keeps its states in registers, so that the sum over the states is
// a chain of FMAs in the lane, and a wave's 64 channels are one run of each token's row. B_t and
// C_t are the same for all of a wave's channels: a first launch writes them as float32 rows
// (`bc`), which the scan then reads through the scalar cache, into scalar registers that the FMAs
// take directly. Neither a shuffle nor LDS is left in the forward's loop; it is bound by the
// vector units: an exponential, two products and two FMAs a state and token. Measured costs of a
// wave's operation in cycles of its SIMD: exponential 8, one with a scalar operand 4, any other 2.
// MI355X, B2 T4096 D4096 N16 bf16: 161 us the outputs with the states kept for the backward (3.3 T
// state steps a second; vector units active 82 % of the time as the counter has it, four cycles for
// any operation but the exponential; 58 % at the costs above); four lanes a channel with B, C
// and delta' in LDS took 204.
//
// Pieces: h_t = a_t h_{t-1} + b_t is linear, so a sequence is cut into pieces that run in
// parallel. A first pass finds each piece's state from zero (L) and its summed delta' (S), a
// small one folds them in order, h <- exp(A S_j) h + L_j, and leaves every piece's entry state
// (at the sizes above 114 us and 18 us: the price of 8192 waves instead of 128).
#include <type_traits>

#include "common.hpp"
#include "ssm.hpp"

namespace tops {

namespace {

constexpr int SS_K = 8;      // tokens of a tile of the backward, and between the states kept for it
constexpr int FT = 4;        // tokens of a tile of the forward
constexpr float kLn2 = 0.6931471805599453f;

// Wave-uniform data that no kernel of the launch writes: read by scalar loads.
typedef const float __attribute__((address_space(4))) cfloat;
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

struct Piece {
  int seq, t0, t1, idx, np, c0;
  long b;
};

__device__ __forceinline__ Piece piece_of(const ScanParams& p, int i) {
  Piece r;
  if (p.a.segs) {
    const int* s = p.a.segs + 8L * i;
    r.seq = uni(s[0]), r.t0 = uni(s[1]), r.t1 = uni(s[2]), r.idx = uni(s[3]), r.np = uni(s[4]);
    r.c0 = uni(s[5]);
    r.b = 0;
  } else {
    const int T = (int)p.a.T, len = (int)p.a.piece;
    r.np = p.pieces;
    r.seq = i / r.np;
    r.idx = i - r.seq * r.np;
    r.t0 = r.idx * len;
    r.t1 = r.t0 + min(T - r.t0, len);   // t0 + len may pass 32 bits
    r.c0 = r.seq * ((T + SS_K - 1) / SS_K) + r.t0 / SS_K;
    r.b = r.seq;
  }
  return r;
}

// A channel tile of 64: its group, first channel, and the lane's channel (the first one where the
// lane has none).
struct Tile {
  int grp, d0, nch;
  __device__ __forceinline__ Tile(const ScanParams& p, int tile) {
    const int DG = (int)(p.a.D / p.a.G);
    grp = tile / p.tiles_g;
    const int cb = (tile - grp * p.tiles_g) * 64;
    d0 = grp * DG + cb;
    nch = min(64, DG - cb);
  }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Keeps the compiler from moving LDS reads up, into registers that others need.
__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }

// The N states of a lane's channel, in rows of D channels.
template <int N>
__device__ __forceinline__ void load_states(const float* p, int D, uint32_t lo, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i, p += D) x[i] = p[lo];
}
template <int N>
__device__ __forceinline__ void store_states(float* p, int D, uint32_t lo, const float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i, p += D) p[lo] = x[i];
}

// The lane's element of N rows from `t` on, the last one of the piece again past its end (t < t1).
template <typename T, int N>
__device__ __forceinline__ void load_rows(const T* p, long st, int t, int t1, uint32_t lo,
                                          T (&x)[N]) {
  p += t * st;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = p[lo];
    p += t + i + 1 < t1 ? st : 0;
  }
}

// A row of bc once the states x are there: the scalar loads of all tokens would otherwise be
// moved to the tile's start, where there are not enough scalar registers for them.
template <int N>
__device__ __forceinline__ cfloat* row_after(const float* p, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile(""
                 : "+s"(p), "+v"(x[i]), "+v"(x[i + 1]), "+v"(x[i + 2]), "+v"(x[i + 3]),
                   "+v"(x[i + 4]), "+v"(x[i + 5]), "+v"(x[i + 6]), "+v"(x[i + 7]));
  return (cfloat*)(uintptr_t)p;
}

// The states that fill N up to 8, 16, 32 or 64 are zero: their B and C are, and A as well. But an
// infinite input times their B is a NaN, which would reach the sums: they are set to zero again
// wherever the lanes' x are not all finite, in kernels of their own (PAD).
__device__ __forceinline__ bool any_odd(float x) { return __any(!(fabsf(x) <= 3.4028235e38f)); }
template <int N>
__device__ __forceinline__ void clear_pads(float (&h)[N], int real) {
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (n >= real) h[n] = 0.f;
}

// Has x computed here: the compiler would put sums off and keep their terms in registers.
__device__ __forceinline__ void pin(float (&x)[8]) {
  asm volatile(""
               : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]),
                 "+v"(x[6]), "+v"(x[7]));
}

// Eight floats of a row, in eight scalar registers in a row as a scalar load leaves them.
typedef float row8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ row8 load_row(cfloat* p) {
  return *(const row8 __attribute__((address_space(4)))*)p;
}
// Waits here for them.
__device__ __forceinline__ void arrived(row8& x) { asm volatile("" : "+s"(x)); }

// B and C as float32 rows [token][group][2][NP], zeros past N and in one more row, which stands
// for the tokens past a piece's end; then A log2(e) as rows of D channels [NP][D].
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_bc_kernel(ScanParams p) {
  const long rows = p.tokens * p.a.G, nbc = (rows + 1) * 2 * NP, total = nbc + p.a.D * NP;
  const int N = (int)p.a.N, G = (int)p.a.G;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const int n = (int)(i % NP), w = (int)(i / NP % 2);
    const long r = i / (2 * NP);
    const int tok = G == 1 ? (int)r : (int)(r / G);   // B T < 2^31
    const long g = r - (long)tok * G;
    if (r >= rows) {
      const int j = (int)(i - nbc), m = j >= 0 ? j / (int)p.a.D : N;   // D NP <= 2^26
      p.a.bc[i] = m < N ? scaled_a(p.a.A[(j - m * (int)p.a.D) * (long)N + m]) : 0.f;
      continue;
    }
    const long b = p.a.batch == 1 ? 0 : tok / (int)p.a.T, t = tok - b * p.a.T;
    const T* s = w ? (const T*)p.a.C + b * p.a.C_sb + t * p.a.C_st + g * p.a.C_sg
                   : (const T*)p.a.B + b * p.a.B_sb + t * p.a.B_st + g * p.a.B_sg;
    p.a.bc[i] = n < N ? to_f32(s[n]) : 0.f;
  }
}

// ---------------------------------------------------------------------------
// A wave walks a piece for 64 channels. MODE 0: a piece's own state and summed delta'. MODE 1:
// the outputs. MODE 2: the reverse of 0 for the backward, the carry that a piece hands to the one
// before it, from a zero carry. PAD: N < NP (MODE 1).
// ---------------------------------------------------------------------------
template <typename T, int NP, int MODE, bool PAD>
__global__ __launch_bounds__(256, NP <= 16 ? 4 : NP <= 32 ? 3 : 2) void scan_kernel(ScanParams p) {
  const tops_gla_scan_args& a = p.a;
  const int lane = threadIdx.x & 63;
  const long item = blockIdx.x * 4L + uni(threadIdx.x >> 6);
  if (item >= p.npieces * p.ntiles) return;
  const int pi = uni((int)(item / p.ntiles));
  const Tile tl(p, uni((int)(item - (long)pi * p.ntiles)));
  const Piece pc = piece_of(p, pi);
  if (MODE == 0 && pc.idx == pc.np - 1) return;   // nobody folds it
  if (MODE == 2 && pc.idx == 0) return;
  const int D = (int)a.D, N = (int)a.N;
  const bool live = lane < tl.nch;
  const uint32_t lo = live ? lane : 0;
  const long dl = tl.d0 + lo;

  constexpr int GN = NP < 16 ? NP : 16;   // states whose rows are in scalar registers at a time
  float A[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = 0.f;
  load_states<NP>(p.at + tl.d0, D, lo, A);
  if (MODE == 1) {
    if (p.multi) {
      load_states<NP>(a.piece_h + (long)pi * NP * D + tl.d0, D, lo, h);
    } else if (a.h0) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (n < N) h[n] = a.h0[((long)pc.seq * D + dl) * N + n];
    }
  }
  const float bias = a.delta_bias ? a.delta_bias[dl] : 0.f;
  const float skip = MODE == 1 && a.Dskip ? a.Dskip[dl] : 0.f;
  const bool has_z = MODE != 0 && a.z != nullptr, softplus = a.softplus;
  float dsum = 0.f;

  // rows of the tensors: uniform addresses, a lane's offset of 32 bits
  const T* gu = MODE == 2 ? (const T*)a.dy + pc.b * a.dy_sb + tl.d0
                          : (const T*)a.u + pc.b * a.u_sb + tl.d0;
  const long u_st = MODE == 2 ? a.dy_st : a.u_st;
  const T* gd = (const T*)a.delta + pc.b * a.delta_sb + tl.d0;
  const T* gz = has_z ? (const T*)a.z + pc.b * a.z_sb + tl.d0 : nullptr;
  const long bc_st = a.G * 2 * NP;
  const float* bc = a.bc + (pc.b * a.T * a.G + tl.grp) * 2 * NP + (MODE == 2 ? NP : 0);
  const float* bc_end = a.bc + p.tokens * bc_st;

  T ru[FT], rd[FT], rz[FT];
  auto load = [&](int t0) {
    load_rows<T, FT>(gu, u_st, t0, pc.t1, lo, ru);
    load_rows<T, FT>(gd, a.delta_st, t0, pc.t1, lo, rd);
    if (has_z) load_rows<T, FT>(gz, a.z_st, t0, pc.t1, lo, rz);
  };
  const int nt = (pc.t1 - pc.t0 + FT - 1) / FT;
  const int first = MODE == 2 ? nt - 1 : 0, step = MODE == 2 ? -1 : 1;
  if (nt > 0) load(pc.t0 + first * FT);
#pragma unroll 1
  for (int it = 0; it < nt; ++it) {
    const int k = first + it * step, t0 = pc.t0 + k * FT;
    float d[FT], u[FT], z[FT], y[FT];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      d[i] = to_f32(rd[i]) + bias;
      u[i] = to_f32(ru[i]);
      z[i] = has_z ? to_f32(rz[i]) : 0.f;
    }
    if (softplus)
#pragma unroll
      for (int i = 0; i < FT; ++i) d[i] = tops::softplus(d[i]);
    if (MODE == 2 && has_z)
#pragma unroll
      for (int i = 0; i < FT; ++i) u[i] *= z[i] * sigmoid(z[i]);
    if (t0 + FT > pc.t1)
#pragma unroll
      for (int i = 0; i < FT; ++i)   // a token past the end leaves the state as it is
        if (t0 + i >= pc.t1) d[i] = u[i] = 0.f;
    if (it + 1 < nt) load(t0 + step * FT);
    if (MODE == 1 && k % (SS_K / FT) == 0 && a.chunk_h && live)
      store_states<NP>(a.chunk_h + (long)(pc.c0 + k / (SS_K / FT)) * NP * D + tl.d0, D, lo, h);
    const float* q = bc + (t0 + (MODE == 2 ? FT - 1 : 0)) * bc_st;
    float ahead[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FT; ++j) {
      const int i = MODE == 2 ? FT - 1 - j : j;
      const float x = MODE == 2 ? u[i] : d[i] * u[i];
      float acc[2] = {0.f, 0.f};
      const float* at = t0 + i < pc.t1 ? q : bc_end;
      q += MODE == 2 ? -bc_st : bc_st;
#pragma unroll
      for (int g = 0; g < NP; g += GN) {
        float(&hg)[GN] = *reinterpret_cast<float(*)[GN]>(&h[g]);
        row8 rb[GN / 8], rc[GN / 8];
        asm volatile("" : : "s"(ahead[0]), "s"(ahead[1]));
        cfloat* row = row_after(at, hg);
#pragma unroll
        for (int i8 = 0; i8 < GN / 8; ++i8) {
          rb[i8] = load_row(row + g + 8 * i8);
          if (MODE == 1) rc[i8] = load_row(row + NP + g + 8 * i8);
        }
#pragma unroll
        for (int i8 = 0; i8 < GN / 8; ++i8) {
          arrived(rb[i8]);
          if (MODE == 1) arrived(rc[i8]);
        }
        const bool more = g + GN < NP;
        if (more || j + 1 < FT) {   // the next rows into the scalar cache
          cfloat* np = more ? row + g + GN
                            : (cfloat*)(uintptr_t)(t0 + i + (MODE == 2 ? -1 : 1) < pc.t1 ? q : bc_end);
          ahead[0] = np[0];
          if (MODE == 1) ahead[1] = np[NP];
        }
#pragma unroll
        for (int n = 0; n < GN; ++n) {
          const float ex = exp2_hw(A[g + n] * d[i]);
          if (MODE == 2) {
            hg[n] = ex * fmaf(x, rb[n / 8][n % 8], hg[n]);
          } else {
            hg[n] = fmaf(ex, hg[n], x * rb[n / 8][n % 8]);
            if (MODE == 1 && !PAD) acc[n & 1] = fmaf(hg[n], rc[n / 8][n % 8], acc[n & 1]);
          }
        }
        if (PAD) {
          if (any_odd(x)) clear_pads<GN>(hg, N - g);
#pragma unroll
          for (int n = 0; n < GN; ++n) acc[n & 1] = fmaf(hg[n], rc[n / 8][n % 8], acc[n & 1]);
        }
        if (MODE == 1) asm volatile("" : "+v"(acc[0]), "+v"(acc[1]));   // like h: now
      }
      y[i] = acc[0] + acc[1];
      if (MODE != 1) dsum += d[i];
    }
    if (MODE == 1) {
      T* gy = (T*)a.y + (pc.b * a.T + t0) * D + tl.d0;
#pragma unroll
      for (int i = 0; i < FT; ++i) y[i] = fmaf(skip, u[i], y[i]);
      if (has_z)
#pragma unroll
        for (int i = 0; i < FT; ++i) y[i] *= z[i] * sigmoid(z[i]);
      if (live)
#pragma unroll
        for (int i = 0; i < FT; ++i)
          if (t0 + i < pc.t1) (gy + (long)i * D)[lo] = from_f32<T>(y[i]);
    }
  }
  if (!live) return;
  if (MODE == 1) {
    if (a.ht && pc.idx == pc.np - 1)
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (n < N) a.ht[((long)pc.seq * D + dl) * N + n] = h[n];
  } else {
    if (N < NP) clear_pads<NP>(h, N);
    store_states<NP>(a.piece_h + (long)pi * NP * D + tl.d0, D, lo, h);
    a.piece_dt[(long)pi * D + dl] = dsum;
  }
}

// The state after a piece of summed delta' s and own state l, entered with h. A zero state stays
// zero under a decay that overflows. An infinite one stays infinite under a decay that is too small
// for a float as the product of its tokens' (2^-126 in its place: nothing to a finite state), but
// not under one that forgets at once (A of -inf).
__device__ __forceinline__ float folded(float h, float A, float s, float l) {
  const float e = A * s, f = exp2_hw(e);
  const float g = e > -1e30f ? fmaxf(f, 1.17549435e-38f) : f;
  return h == 0.f ? l : fmaf(g, h, l);
}

// The pieces' entry states in the place of their own ones: h <- exp(A S_j) h + L_j over a
// sequence's pieces from h0 on, or backward from dht on with REV. A thread folds a run of the
// pieces for a state of a channel, 4 threads share a sequence's runs: each finds its run's own L
// and S, then its entry from those of the runs before, then its pieces' entries. Runs of up to 16
// pieces are read once.
constexpr int FOLD_R = 4, FOLD_U = 16, FOLD_NT = 64 * FOLD_R;
template <int NP, bool REV>
__global__ __launch_bounds__(FOLD_NT) void scan_fold_kernel(ScanParams p) {
  __shared__ float sL[FOLD_R][64], sS[FOLD_R][64];
  const tops_gla_scan_args& a = p.a;
  const long seq = blockIdx.y + (long)blockIdx.z * gridDim.y;
  if (seq >= a.nseq) return;
  const long pi = a.segs ? a.segs[8 * seq + 6] : seq * p.pieces;
  const int np = uni(piece_of(p, (int)pi).np), m = (np + FOLD_R - 1) / FOLD_R;
  const int run = uni(threadIdx.x / 64), c = threadIdx.x % 64;
  const int D = (int)a.D, N = (int)a.N;
  const int n = blockIdx.x % NP, d = blockIdx.x / NP * 64 + c;
  const long nd = (long)D * NP;
  if (d >= D) return;   // the same lanes of every wave: their columns of sL and sS are not used
  const int j0 = min(np, run * m), j1 = min(np, j0 + m);
  const float* init = REV ? a.dht : a.h0;
  const float A = p.at[(long)n * D + d];
  const long first = pi + (REV ? np - 1 : 0);
  const long hs = (REV ? -1L : 1L) * nd, ss = (REV ? -1L : 1L) * D;
  float* H = a.piece_h + first * nd + (long)n * D + d;
  const float* S = a.piece_dt + first * D + d;
  float h = 0.f, s = 0.f;
  float l[FOLD_U], dt[FOLD_U];
  // h through the pieces j .. end - 1, each piece's entry state written with `put`; the last piece
  // has no own state
  auto walk = [&](int j, int end, bool put) {
    for (; j < end; j += FOLD_U) {
      if (!put || m > FOLD_U)
#pragma unroll
        for (int i = 0; i < FOLD_U; ++i) {
          if (j + i >= min(end, np - 1)) break;
          l[i] = H[(j + i) * hs];
          dt[i] = S[(j + i) * ss];
        }
#pragma unroll
      for (int i = 0; i < FOLD_U; ++i) {
        if (j + i >= end) break;
        if (put) H[(j + i) * hs] = h;
        if (j + i < np - 1) {
          h = folded(h, A, dt[i], l[i]);
          s += dt[i];
        }
      }
    }
  };
  walk(j0, j1, false);
  sL[run][c] = h;
  sS[run][c] = s;
  __syncthreads();
  h = n < N && init ? init[(seq * D + d) * N + n] : 0.f;
  for (int r = 0; r < run; ++r) h = folded(h, A, sS[r][c], sL[r][c]);
  walk(j0, j1, true);
}

// ---------------------------------------------------------------------------
// Backward, over a piece's tiles of 8 tokens from the last one on. With g_t the gradient of h_t,
// g_t = C_t dy_t + a_{t+1} g_{t+1}:
//   dC_t = sum_d dy_t h_t          dB_t = sum_d g_t delta' u        du = delta' sum_n g B + D dy
//   ddelta' = u sum_n g B + sum_n g a h_{t-1} A                     dA = sum_t g a h_{t-1} delta'
// A tile's states run forward again from the one that the forward kept, with a_t and h_t of its
// tokens in registers (recovering h_{t-1} from h_t would divide by a_t).
//
// A lane holds 8 states of a channel, the NW = NP / 8 waves of a channel group a part of the
// states each. They share what is formed once for a (token, channel) through LDS: each wave
// stages 8 / NW of the tile's tokens and, once the waves' sums over n are there, finishes them. The
// sums over the channels, of 16 values a token, transpose on their way down (32 operations for
// them all). Bound by vector issue (active 87 % of the time as counted, 53 % at the costs above): 25
// instructions a state and token, 18 of them the formulas'; the compiler moves 60 to 105 scalars to
// lanes of vector registers (82 with 16 states). MI355X, B2 T4096 D4096 N16 bf16: 481 us (a token more in registers costs the third
// wave of a SIMD: all 8 at two waves 574; four lanes a channel and LDS rows of B and C 1145).
//
// EDGE: 1 with padded states, 2 where some lanes have no channel (padded states or not). Infinite
// values must not meet their zeros; the checks cost 1.5 and 3 % of the training pass (B2 T4096, N 12,
// D 4096 and 4000).
// ---------------------------------------------------------------------------
constexpr int HK = SS_K / 2;
// Steps 0 .. 5 HK - 1 of a tile: forward to its middle; the second half forward, and back; the
// first half forward, and back. The token of a step, and whether it goes back.
constexpr bool is_back(int e) { return e / HK == 2 || e / HK == 4; }
constexpr int token_of(int e) {
  return e < 2 * HK   ? e
         : e < 3 * HK ? 4 * HK - 1 - e
         : e < 4 * HK ? e - 3 * HK
                      : 5 * HK - 1 - e;
}
template <int I, int N, typename F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<I + 1, N>(f);
  }
}

template <int NP>
struct Bwd {
  static constexpr int NW = NP / 8;                // waves of a channel group
  static constexpr int WAVES = NP == 64 ? 8 : 4;   // of a block
  static constexpr int GPB = WAVES / NW;           // channel groups (of 64) of a block
  static constexpr int CT = 64 * GPB;
  static constexpr int TPW = SS_K / NW;            // tokens that a wave stages
};

// Level of a transposing sum over the lanes of a row of 16: lanes of the banks that `odd` names
// get b's sum with lane `ctrl`, the others a's. (A DPP or swap operand may be read two wait states
// after it was written; the compiler does not see these writes and reads.)
#define TOPS_PAIR4(ctrl, odd, a0, b0, a1, b1, a2, b2, a3, b3)                                   \
  asm("s_nop 1\n\t"                                                                             \
      "v_add_f32_dpp %0, %0, %0 " ctrl " row_mask:0xf bank_mask:0xf\n\t"                        \
      "v_add_f32_dpp %1, %1, %1 " ctrl " row_mask:0xf bank_mask:0xf\n\t"                        \
      "v_add_f32_dpp %2, %2, %2 " ctrl " row_mask:0xf bank_mask:0xf\n\t"                        \
      "v_add_f32_dpp %3, %3, %3 " ctrl " row_mask:0xf bank_mask:0xf\n\t"                        \
      "v_add_f32_dpp %0, %4, %4 " ctrl " row_mask:0xf bank_mask:" odd "\n\t"                    \
      "v_add_f32_dpp %1, %5, %5 " ctrl " row_mask:0xf bank_mask:" odd "\n\t"                    \
      "v_add_f32_dpp %2, %6, %6 " ctrl " row_mask:0xf bank_mask:" odd "\n\t"                    \
      "v_add_f32_dpp %3, %7, %7 " ctrl " row_mask:0xf bank_mask:" odd "\n\ts_nop 1"              \
      : "+&v"(a0), "+&v"(a1), "+&v"(a2), "+&v"(a3)                                              \
      : "v"(b0), "v"(b1), "v"(b2), "v"(b3))

// x[0..7] and y[0..7] summed over the 64 lanes: lane l ends with element 4 l[2] + 2 l[4] + l[5]
// of x, of y where bit 3 is set (l[i]: bit i of l).
__device__ __forceinline__ float sum_channels(float (&x)[8], float (&y)[8]) {
  TOPS_PAIR4("row_ror:8", "0xc", x[0], y[0], x[1], y[1], x[2], y[2], x[3], y[3]);
  TOPS_PAIR4("row_ror:8", "0xc", x[4], y[4], x[5], y[5], x[6], y[6], x[7], y[7]);
  TOPS_PAIR4("row_half_mirror", "0xa", x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]);
  float s = swap32_add(swap16_add(x[0], x[2]), swap16_add(x[1], x[3]));
  s += dpp<0xb1>(s);      // quad_perm [1, 0, 3, 2]
  return s + dpp<0x4e>(s);   // quad_perm [2, 3, 0, 1]
}

template <typename T, int NP, int EDGE>
__global__ __launch_bounds__(64 * Bwd<NP>::WAVES, NP == 16 || NP == 32 ? 3 : 2) void scan_bwd_kernel(ScanParams p) {
  using L = Bwd<NP>;
  __shared__ float sD[SS_K][L::CT], sU[SS_K][L::CT], sG[SS_K][L::CT];   // delta', u, dy silu(z)
  __shared__ float sK[2][SS_K][L::CT];          // softplus', dy silu'(z): for the wave that staged them
  __shared__ float sS[L::NW][3][SS_K][L::CT];   // sum_n g B, sum_n g a h A log2(e), sum_n C h
  __shared__ float sBC[L::GPB][SS_K][2 * NP];   // a channel group's dB and dC
  const tops_gla_scan_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int part = wave % L::NW, cg = wave / L::NW;
  const int tile = blockIdx.x % p.btiles, pi = blockIdx.x / p.btiles;
  const Piece pc = piece_of(p, pi);
  const int D = (int)a.D, N = (int)a.N, DG = D / (int)a.G;
  const int btiles_g = p.btiles / (int)a.G, grp = tile / btiles_g;
  const int cb = (tile - grp * btiles_g) * L::CT + 64 * cg;   // first channel in its group
  const int d0 = grp * DG + min(cb, DG - 1);
  const bool live = cb + lane < DG;
  const uint32_t lo = live ? lane : 0;
  const long dl = d0 + lo;
  const int n0 = 8 * part, col = 64 * cg + lane;
  const bool pads = EDGE == 1 || (EDGE == 2 && N < NP);
  float A[8], carry[8], dA[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) carry[n] = dA[n] = 0.f;
  load_states<8>(p.at + (long)n0 * D + d0, D, lo, A);
  if (live) {
    if (p.multi) {
      load_states<8>(a.piece_h + ((long)pi * NP + n0) * D + d0, D, lo, carry);
    } else if (a.dht) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
        if (n0 + n < N) carry[n] = a.dht[((long)pc.seq * D + dl) * N + n0 + n];
    }
  }
  const float bias = a.delta_bias ? a.delta_bias[dl] : 0.f;
  const float skip = a.Dskip ? a.Dskip[dl] : 0.f;
  const bool has_z = a.z != nullptr, softplus = a.softplus;
  float accD = 0.f, accB = 0.f;

  const T* gu = (const T*)a.u + pc.b * a.u_sb + d0;
  const T* gd = (const T*)a.delta + pc.b * a.delta_sb + d0;
  const T* gz = has_z ? (const T*)a.z + pc.b * a.z_sb + d0 : nullptr;
  const T* gy = (const T*)a.dy + pc.b * a.dy_sb + d0;
  const float* bc = a.bc + (pc.b * a.T * a.G + grp) * 2 * NP + n0;
  const long bc_st = a.G * 2 * NP;
  const float* bc_end = a.bc + p.tokens * bc_st;
  T ru[L::TPW], rd[L::TPW], rz[L::TPW], ry[L::TPW];
  float rh[8];
  auto load = [&](int k) {
    const int t0 = min(pc.t0 + k * SS_K + part * L::TPW, pc.t1 - 1);
    load_rows<T, L::TPW>(gu, a.u_st, t0, pc.t1, lo, ru);
    load_rows<T, L::TPW>(gd, a.delta_st, t0, pc.t1, lo, rd);
    load_rows<T, L::TPW>(gy, a.dy_st, t0, pc.t1, lo, ry);
    if (has_z) load_rows<T, L::TPW>(gz, a.z_st, t0, pc.t1, lo, rz);
    load_states<8>(a.chunk_h + ((long)(pc.c0 + k) * NP + n0) * D + d0, D, lo, rh);
  };
  const int nt = (pc.t1 - pc.t0 + SS_K - 1) / SS_K;
  if (nt > 0) load(nt - 1);
#pragma unroll 1
  for (int k = nt - 1; k >= 0; --k) {
    const int t0 = pc.t0 + k * SS_K, ts = part * L::TPW;
    float sd[L::TPW], sg[L::TPW];
#pragma unroll
    for (int i = 0; i < L::TPW; ++i) sd[i] = to_f32(rd[i]) + bias, sg[i] = 1.f;
    if (softplus)
#pragma unroll
      for (int i = 0; i < L::TPW; ++i) softplus_sigmoid(sd[i], sd[i], sg[i]);
#pragma unroll
    for (int i = 0; i < L::TPW; ++i) {
      const bool in = live && t0 + ts + i < pc.t1;
      const float d = sd[i];
      const float dy = to_f32(ry[i]), z = has_z ? to_f32(rz[i]) : 0.f;
      const float sz = sigmoid(z), g = has_z ? dy * z * sz : dy;
      sK[0][ts + i][col] = sg[i];
      sK[1][ts + i][col] = dy * (sz * fmaf(z, 1.f - sz, 1.f));   // dy silu'(z)
      sD[ts + i][col] = in ? d : 0.f;
      sU[ts + i][col] = in ? to_f32(ru[i]) : 0.f;
      sG[ts + i][col] = in ? g : 0.f;
    }
    float hin[8], hm[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) hin[n] = hm[n] = live ? rh[n] : 0.f;
    // Three sweeps over four tokens at a time: the first half's states forward without keeping
    // them, then each half, the second one first, forward with a_t and h_t in registers and back.
    // The rows of a token are fetched while the one before it is computed: B and C into scalar
    // registers, delta', u and dy from LDS. One counter stands for both kinds of loads, and the
    // scalar ones come in any order: a wait has to be for all of them, before the next are sent.
    const float* rows = bc + t0 * bc_st;
    float nd, nu, ng, av[HK][8], hv[HK][8];
    row8 nb = load_row(row_after(rows, hin)), nc;
    __syncthreads();
    nd = sD[0][col];
    nu = sU[0][col];
    static_for<0, 5 * HK>([&](auto step) {
      constexpr int e = decltype(step)::value, sweep = e / HK;
      constexpr bool back = is_back(e), nback = is_back(e + 1);
      constexpr int t = token_of(e), tn = token_of(e + 1), s = t % HK;
      float(&h0)[8] = sweep < 3 ? hm : hin;
      arrived(nb);
      asm volatile("" : "+v"(nd), "+v"(nu));
      if constexpr (back) {
        arrived(nc);
        asm volatile("" : "+v"(ng));
      }
      const row8 rb = nb, rc = nc;
      const float d = nd, x = d * nu, dy = ng;
      if constexpr (e + 1 < 5 * HK) {
        const float* at = t0 + tn < pc.t1 ? rows + tn * bc_st : bc_end;
        cfloat* row;
        if constexpr (back)
          row = row_after(at, carry);
        else if constexpr (sweep == 0 || s == 0)
          row = row_after(at, h0);
        else
          row = row_after(at, hv[s - 1]);
        nb = load_row(row);
        if (nback) nc = load_row(row + NP);
        nd = sD[tn][col];
        nu = sU[tn][col];
        if (nback) ng = sG[tn][col];
      }
      if (e == 3 * HK && k > 0) load(k - 1);
      if constexpr (sweep == 0) {
#pragma unroll
        for (int n = 0; n < 8; ++n) hm[n] = fmaf(exp2_hw(A[n] * d), hm[n], x * rb[n]);
        if (pads && any_odd(x)) clear_pads<8>(hm, N - n0);
      } else if constexpr (!back) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          av[s][n] = exp2_hw(A[n] * d);
          if constexpr (s > 0)
            hv[s][n] = fmaf(av[s][n], hv[s - 1][n], x * rb[n]);
          else
            hv[s][n] = fmaf(av[s][n], h0[n], x * rb[n]);
        }
        if (pads && any_odd(x)) {
          clear_pads<8>(av[s], N - n0);   // 0 times an infinite delta'
          clear_pads<8>(hv[s], N - n0);
        }
      } else {
        float vb[8], vc[8], gd[8], s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int n = 0; n < 8; ++n) carry[n] = fmaf(dy, rc[n], carry[n]);
        if (pads && any_odd(dy)) clear_pads<8>(carry, N - n0);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float g = carry[n];
          float hp = h0[n];
          if constexpr (s > 0) hp = hv[s - 1][n];
          vb[n] = g * x;
          vc[n] = dy * hv[s][n];
          s1 = fmaf(g, rb[n], s1);
          carry[n] = av[s][n] * g;
          const float gp = carry[n] * hp;
          s2 = fmaf(gp, A[n], s2);
          s3 = fmaf(hv[s][n], rc[n], s3);
          gd[n] = gp;
        }
        if (t0 + t < pc.t1)   // past the end 0 times a state, which an infinity makes NaN
#pragma unroll
          for (int n = 0; n < 8; ++n) dA[n] = fmaf(gd[n], d, dA[n]);
        pin(dA);
        sS[part][0][t][col] = s1;
        sS[part][1][t][col] = s2;
        sS[part][2][t][col] = s3;
        if (EDGE == 2 && cb + 64 > DG)   // lanes without a channel: zeros, but not times an infinite B or C
#pragma unroll
          for (int n = 0; n < 8; ++n) vb[n] = live ? vb[n] : 0.f, vc[n] = live ? vc[n] : 0.f;
        const float r = sum_channels(vb, vc);
        if ((lane & 3) == 0)
          sBC[cg][t][(lane & 8 ? NP : 0) + n0 + (lane & 4) + ((lane >> 3) & 2) + (lane >> 5)] = r;
        fence();
      }
    });
    __syncthreads();
    const long o = (pc.b * a.T + t0 + ts) * D + d0;
    T *odu = (T*)a.du + o, *odd = (T*)a.ddelta + o, *odz = (T*)a.dz + o;
#pragma unroll
    for (int i = 0; i < L::TPW; ++i) {
      const int t = ts + i;
      float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int w = 0; w < L::NW; ++w) {
        s1 += sS[w][0][t][col];
        s2 += sS[w][1][t][col];
        s3 += sS[w][2][t][col];
      }
      const float d = sD[t][col], u = sU[t][col], dy = sG[t][col];
      const float du = fmaf(s1, d, skip * dy), dd = fmaf(s1, u, s2 * kLn2) * sK[0][t][col];
      const float dz = sK[1][t][col] * fmaf(skip, u, s3);
      if (live && t0 + t < pc.t1) {
        accD = fmaf(dy, u, accD);
        accB += dd;
        odu[lo] = from_f32<T>(du);
        odd[lo] = from_f32<T>(dd);
        if (has_z) odz[lo] = from_f32<T>(dz);
      }
      odu += D;
      odd += D;
      odz += D;
    }
    // the block's share of dB and dC: [tile of the group][token][group][2][NP]
    for (int i = tid; i < SS_K * 2 * NP; i += 64 * L::WAVES) {
      const int t = i / (2 * NP), c = i % (2 * NP);
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < L::GPB; ++w) s += sBC[w][t][c];
      if (t0 + t < pc.t1)
        p.part_bc[(((long)(tile - grp * btiles_g) * p.tokens + pc.b * a.T + t0 + t) * a.G + grp) *
                      (2 * NP) + c] = s;
    }
    // sD, sU and sG are written next by the wave that read them here; sS and sBC after a barrier
  }
  if (live) {
    if (pc.idx == 0 && a.dh0)
#pragma unroll
      for (int n = 0; n < 8; ++n)
        if (n0 + n < N) a.dh0[((long)pc.seq * D + dl) * N + n0 + n] = carry[n];
    store_states<8>(p.part_a + ((long)pi * NP + n0) * D + d0, D, lo, dA);
  }
  // dD and the bias: sum over the waves of a channel group
  __syncthreads();
  sS[part][0][0][col] = accD;
  sS[part][1][0][col] = accB;
  __syncthreads();
  if (part == 0 && live) {
    float sd = 0.f, sb = 0.f;
#pragma unroll
    for (int w = 0; w < L::NW; ++w) {
      sd += sS[w][0][0][col];
      sb += sS[w][1][0][col];
    }
    p.part_d[(long)pi * 2 * D + dl] = sd;
    p.part_d[((long)pi * 2 + 1) * D + dl] = sb;
  }
}

// dB, dC from the blocks' shares: one thread per (token, group, array, n).
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_bwd_bc_kernel(ScanParams p) {
  const long total = p.tokens * p.a.G * 2 * NP;
  const int N = (int)p.a.N, tiles = p.btiles / (int)p.a.G;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    float s = 0.f;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) s += p.part_bc[t * total + i];
    const int c = (int)(i % (2 * NP)), n = c % NP;
    if (n < N) ((T*)(c < NP ? p.a.dB : p.a.dC))[(i / (2 * NP)) * N + n] = from_f32<T>(s);
  }
}

// dA, dD, dbias from the pieces' shares, 8 threads a column.
__global__ __launch_bounds__(256) void scan_bwd_a_kernel(ScanParams p, int NP) {
  __shared__ float red[8][32];
  const long D = p.a.D, na = D * NP;
  const int N = (int)p.a.N, row = threadIdx.x / 32, c = threadIdx.x % 32;
  const long i = blockIdx.x * 32L + c;
  const bool isa = i < na, in = i < na + 2 * D;
  const float* src = isa ? p.part_a + i : p.part_d + (i - na);
  const long st = isa ? na : 2 * D;
  float s = 0.f;
  if (in)
#pragma unroll 8
    for (long j = row; j < p.npieces; j += 8) s += src[j * st];
  red[row][c] = s;
  __syncthreads();
  if (row || !in) return;
  s = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) s += red[r][c];
  if (isa) {
    const int n = (int)i / (int)D;   // D NP <= 2^26
    const long d = i - n * D;
    if (n < N) p.a.dA[d * N + n] = s;
  } else {
    const long r = i - na;
    float* out = r < D ? p.a.dD : p.a.dbias;
    if (out) out[r % D] = s;
  }
}

unsigned grid_of(long threads) {
  return (unsigned)std::min<long>((threads + 255) / 256, 1L << 20);
}

template <int NP, bool REV>
hipError_t scan_fold(const ScanParams& p, hipStream_t st) {
  // a sequence in y and z: all in x, many packed sequences would be 2^32 threads and more
  const unsigned y = (unsigned)std::clamp<long>(p.a.nseq, 1, 65535);
  const dim3 grid((unsigned)((p.a.D + 63) / 64 * NP), y, (unsigned)((p.a.nseq + y - 1) / y));
  hipLaunchKernelGGL((scan_fold_kernel<NP, REV>), grid, dim3(FOLD_NT), 0, st, p);
  return hipGetLastError();
}

template <typename T, int NP>
hipError_t scan_fwd(const ScanParams& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.npieces * p.ntiles + 3) / 4));
  const long nbc = (p.tokens * p.a.G + 1) * 2 * NP + p.a.D * NP;
  hipLaunchKernelGGL((scan_bc_kernel<T, NP>), dim3(grid_of(nbc)), dim3(256), 0, st, p);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.multi) {
    hipLaunchKernelGGL((scan_kernel<T, NP, 0, false>), grid, dim3(256), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
    if (hipError_t e = scan_fold<NP, false>(p, st)) return e;
  }
  if (p.a.N < NP)
    hipLaunchKernelGGL((scan_kernel<T, NP, 1, true>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((scan_kernel<T, NP, 1, false>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

template <typename T, int NP>
hipError_t scan_bwd(const ScanParams& p, hipStream_t st) {
  if (p.multi) {
    const dim3 grid((unsigned)((p.npieces * p.ntiles + 3) / 4));
    hipLaunchKernelGGL((scan_kernel<T, NP, 2, false>), grid, dim3(256), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
    if (hipError_t e = scan_fold<NP, true>(p, st)) return e;
  }
  if (p.npieces > 0) {
    const dim3 bgrid((unsigned)(p.npieces * p.btiles)), nt(64 * Bwd<NP>::WAVES);
    if (p.a.D / p.a.G % Bwd<NP>::CT)
      hipLaunchKernelGGL((scan_bwd_kernel<T, NP, 2>), bgrid, nt, 0, st, p);
    else if (p.a.N < NP)
      hipLaunchKernelGGL((scan_bwd_kernel<T, NP, 1>), bgrid, nt, 0, st, p);
    else
      hipLaunchKernelGGL((scan_bwd_kernel<T, NP, 0>), bgrid, nt, 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  const long nbc = p.tokens * p.a.G * 2 * NP, na = p.a.D * (NP + 2);
  if (nbc > 0) {
    hipLaunchKernelGGL((scan_bwd_bc_kernel<T, NP>), dim3(grid_of(nbc)), dim3(256), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  hipLaunchKernelGGL(scan_bwd_a_kernel, dim3((unsigned)((na + 31) / 32)), dim3(256), 0, st, p, NP);
  return hipGetLastError();
}

template <typename T>
hipError_t scan_any(const ScanParams& p, bool backward, hipStream_t st) {
  switch (scan_state_pad((int)p.a.N)) {
    case 8: return backward ? scan_bwd<T, 8>(p, st) : scan_fwd<T, 8>(p, st);
    case 16: return backward ? scan_bwd<T, 16>(p, st) : scan_fwd<T, 16>(p, st);
    case 32: return backward ? scan_bwd<T, 32>(p, st) : scan_fwd<T, 32>(p, st);
    default: return backward ? scan_bwd<T, 64>(p, st) : scan_fwd<T, 64>(p, st);
  }
}

}  // namespace

int scan_state_pad(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }
int scan_chunk() { return SS_K; }
int scan_bwd_threads(int N) { return scan_state_pad(N) == 64 ? 64 * Bwd<64>::WAVES : 64 * Bwd<32>::WAVES; }
int scan_bwd_channels(int N) {
  switch (scan_state_pad(N)) {
    case 8: return Bwd<8>::CT;
    case 16: return Bwd<16>::CT;
    case 32: return Bwd<32>::CT;
    default: return Bwd<64>::CT;
  }
}

hipError_t run_selective_scan(const ScanParams& p, bool backward, hipStream_t st) {
  if (p.a.D == 0 || (p.npieces == 0 && !backward)) return hipSuccess;
  return p.a.dtype == DT_BF16 ? scan_any<bf16>(p, backward, st) : scan_any<float>(p, backward, st);
}

}  // namespace tops
