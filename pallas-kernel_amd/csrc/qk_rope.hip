// Norms of queries and keys for each head with the position rotation in the same pass, forward
// and backward (include/tops_gla_ssm.h).
//
// Bound by memory: a head's row is read and written once. LPR lanes hold a row, VEC elements each,
// so that its mean square is a sum over LPR lanes; a rotated element's partner comes from its lane.
// cos and sin of a token's angles are formed once for all its heads, in LDS: the angle is taken in
// turns in 64 bits, where a far position times a frequency keeps its fraction, and only the fraction
// is rounded to 32. MI355X, B4 T8192 H16+16 D128 bf16: forward 112 us (4.7 TB/s), backward 164 (4.9).
//
// The first two kernels, an element (or, for rows of more than 64 pieces, a piece of four) a lane and
// the partner read again, take what is left: heads of an odd size, rows at odd addresses, and above
// 128 columns those whose size or, in the half layout, rotated half is no multiple of four.
#include "ssm.hpp"

namespace tops {

namespace {

constexpr int QK_NT = 256;
constexpr int QK_MAXTB = 16;   // most tokens whose angles a block forms at a time

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  if constexpr (LPR >= 2) x += dpp<0xb1>(x);
  if constexpr (LPR >= 4) x += dpp<0x4e>(x);
  if constexpr (LPR >= 8) x += dpp<0x141>(x);
  if constexpr (LPR >= 16) x += dpp<0x140>(x);
  if constexpr (LPR >= 32) x = swap16_add(x, x);
  if constexpr (LPR >= 64) x = swap32_add(x, x);
  return x;
}

// VEC elements of a row from column c, `nv` of them valid.
template <typename T, int VEC>
__device__ __forceinline__ void row_load(const T* p, int nv, float (&x)[VEC]) {
  if constexpr (VEC > 1) {
    struct alignas(VEC * sizeof(T)) Raw { T v[VEC]; };
    if (nv > 0) {   // whole or nothing
      const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = to_f32(r.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = 0.f;
    }
  } else {
    x[0] = nv > 0 ? to_f32(p[0]) : 0.f;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void row_store(T* p, int nv, const float (&x)[VEC]) {
  if (nv <= 0) return;
  if constexpr (VEC > 1) {
    store_run<T, VEC>(p, x);
  } else {
    p[0] = from_f32<T>(x[0]);
  }
}

// cos and sin of the angles of tokens tau0 .. tau0 + nt, for all threads of the block.
__device__ __forceinline__ void angles(const tops_gla_qk_args& a, long tau0, int nt, float2* cs) {
  const int R2 = (int)a.R / 2;
  for (int i = threadIdx.x; i < nt * R2; i += QK_NT) {
    const int k = i / R2, f = i - k * R2;
    const uint32_t tau = (uint32_t)(tau0 + k), b = tau / (uint32_t)a.T, t = tau - b * (uint32_t)a.T;
    long pos = t;
    if (a.positions) {
      const long at = (long)b * a.pos_sb + t;
      pos = a.pos64 ? (long)((const int64_t*)a.positions)[at]
                    : (long)((const int32_t*)a.positions)[at];
    }
    // half turns: pos inv_freq / pi, less the nearest even number
    const double h = (double)pos * (a.inv_freq[f] * 0.31830988618379067154);
    const float r = (float)(h - 2.0 * rint(0.5 * h));
    float s, c;
    sincospif(r, &s, &c);
    cs[i] = make_float2(c, s);
  }
}

// One lane's view of a row: NI pieces of VEC columns, LPR * VEC apart, with the columns' partners.
template <int VEC, int LPR, int NI, bool INTER>
struct Cols {
  int c[NI], pc[NI], f[NI], nv[NI];   // column, partner's column, frequency, valid elements
  bool rot[NI], hi[NI];               // VEC > 1, or not interleaved: whole pieces
  __device__ __forceinline__ void init(int lane, int D, int R) {
    const int R2 = R / 2;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      c[j] = (lane + LPR * j) * VEC;
      nv[j] = min(VEC, D - c[j]);
      rot[j] = nv[j] > 0 && c[j] < R;
      if (INTER) {
        hi[j] = c[j] & 1;   // VEC == 1
        pc[j] = VEC > 1 ? c[j] : c[j] ^ 1;
        f[j] = c[j] / 2;
      } else {
        hi[j] = c[j] >= R2;
        pc[j] = hi[j] ? c[j] - R2 : c[j] + R2;
        f[j] = hi[j] ? c[j] - R2 : c[j];
      }
      if (!rot[j]) pc[j] = c[j], f[j] = 0;
    }
  }
};

// x turned by its angles (sign -1: back); xp: the partners' values (unused when pairs are whole).
template <int VEC, bool INTER>
__device__ __forceinline__ void turn(float (&x)[VEC], const float (&xp)[VEC], const float2* cs,
                                     bool rot, bool hi, int c, int R, float sign) {
  if (!rot) return;
  if constexpr (INTER && VEC > 1) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      if (c + e < R) {
        const float2 k = cs[e / 2];
        const float s = sign * k.y, a = x[e], b = x[e + 1];
        x[e] = a * k.x - b * s;
        x[e + 1] = b * k.x + a * s;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float2 k = cs[e];
      const float s = hi ? sign * k.y : -sign * k.y;
      x[e] = fmaf(xp[e], s, x[e] * k.x);
    }
  }
}

template <typename T, int VEC, int LPR, int NI, bool INTER>
__global__ __launch_bounds__(QK_NT) void qk_fwd_kernel(tops_gla_qk_args a, int tb) {
  extern __shared__ float2 cs[];
  const int lane = threadIdx.x % LPR, row0 = threadIdx.x / LPR;
  constexpr int RPB = QK_NT / LPR;
  const int D = (int)a.D, R = (int)a.R, R2 = R / 2;
  const long tokens = a.batch * a.T, tau0 = (long)blockIdx.x * tb;
  const int nt = (int)min((long)tb, tokens - tau0);
  Cols<VEC, LPR, NI, INTER> k;
  k.init(lane, D, R);
  angles(a, tau0, nt, cs);
  __syncthreads();
  const float inv_d = 1.f / (float)D, eps = (float)a.eps;
  constexpr bool PAIR = !(INTER && VEC > 1);   // partners in another piece
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const int H = (int)(part ? a.Hk : a.Hq);
    const T* src = (const T*)(part ? a.k : a.q);
    T* dst = (T*)(part ? a.ko : a.qo);
    const float* w = part ? a.kw : a.qw;
    const long sb = part ? a.k_sb : a.q_sb, st = part ? a.k_st : a.q_st,
               sh = part ? a.k_sh : a.q_sh;
    float wv[NI][VEC], wp[NI][VEC];
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        wv[j][e] = w && e < k.nv[j] ? w[k.c[j] + e] : 1.f;
        if (PAIR) wp[j][e] = w && k.rot[j] ? w[k.pc[j] + e] : 1.f;
      }
    for (int r = row0; r < nt * H; r += RPB) {
      const int tk = r / H, hd = r - tk * H;
      const long tau = tau0 + tk, b = tau / a.T, t = tau - b * a.T;
      const T* x = src + b * sb + t * st + hd * sh;
      T* y = dst + (tau * H + hd) * D;
      float v[NI][VEC], p[NI][VEC], ss = 0.f;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        row_load<T, VEC>(x + (k.nv[j] > 0 ? k.c[j] : 0), k.nv[j], v[j]);
        if (PAIR) row_load<T, VEC>(x + k.pc[j], k.rot[j] ? VEC : 0, p[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss = fmaf(v[j][e], v[j][e], ss);
      }
      const float rstd = rsqrtf(fmaf(row_sum<LPR>(ss), inv_d, eps));
#pragma unroll
      for (int j = 0; j < NI; ++j) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[j][e] *= rstd * wv[j][e];
          if (PAIR) p[j][e] *= rstd * wp[j][e];
        }
        turn<VEC, INTER>(v[j], p[j], cs + tk * R2 + k.f[j], k.rot[j], k.hi[j], k.c[j], R, 1.f);
        row_store<T, VEC>(y + k.c[j], k.nv[j], v[j]);
      }
    }
  }
}

// d: the output's gradient turned back; m = x rstd. dw = sum d m; with e = d w:
// dx = rstd (e - m mean(e m)).
template <typename T, int VEC, int LPR, int NI, bool INTER>
__global__ __launch_bounds__(QK_NT) void qk_bwd_kernel(tops_gla_qk_args a, long ngroups, int tb,
                                                       float* part_w) {
  extern __shared__ float2 cs[];
  __shared__ float red[QK_NT * VEC];
  const int lane = threadIdx.x % LPR, row0 = threadIdx.x / LPR;
  constexpr int RPB = QK_NT / LPR;
  const int D = (int)a.D, R = (int)a.R, R2 = R / 2;
  const long tokens = a.batch * a.T;
  Cols<VEC, LPR, NI, INTER> k;
  k.init(lane, D, R);
  const float inv_d = 1.f / (float)D, eps = (float)a.eps;
  constexpr bool PAIR = !(INTER && VEC > 1);
  float dw[2][NI][VEC] = {};
  for (long g = blockIdx.x; g < ngroups; g += gridDim.x) {
    const long tau0 = g * tb;
    const int nt = (int)min((long)tb, tokens - tau0);
    __syncthreads();
    angles(a, tau0, nt, cs);
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int H = (int)(part ? a.Hk : a.Hq);
      const T* src = (const T*)(part ? a.k : a.q);
      const T* gsrc = (const T*)(part ? a.dko : a.dqo);
      T* dst = (T*)(part ? a.dk : a.dq);
      const float* w = part ? a.kw : a.qw;
      const long sb = part ? a.k_sb : a.q_sb, st = part ? a.k_st : a.q_st,
                 sh = part ? a.k_sh : a.q_sh;
      const long gb = part ? a.dk_sb : a.dq_sb, gt = part ? a.dk_st : a.dq_st,
                 gh = part ? a.dk_sh : a.dq_sh;
      float wv[NI][VEC];
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) wv[j][e] = w && e < k.nv[j] ? w[k.c[j] + e] : 1.f;
      for (int r = row0; r < nt * H; r += RPB) {
        const int tk = r / H, hd = r - tk * H;
        const long tau = tau0 + tk, b = tau / a.T, t = tau - b * a.T;
        const T* x = src + b * sb + t * st + hd * sh;
        const T* gy = gsrc + b * gb + t * gt + hd * gh;
        float v[NI][VEC], d[NI][VEC], p[NI][VEC], ss = 0.f, em = 0.f;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int c = k.nv[j] > 0 ? k.c[j] : 0;
          row_load<T, VEC>(x + c, k.nv[j], v[j]);
          row_load<T, VEC>(gy + c, k.nv[j], d[j]);
          if (PAIR) row_load<T, VEC>(gy + k.pc[j], k.rot[j] ? VEC : 0, p[j]);
          turn<VEC, INTER>(d[j], p[j], cs + tk * R2 + k.f[j], k.rot[j], k.hi[j], k.c[j], R, -1.f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            ss = fmaf(v[j][e], v[j][e], ss);
            em = fmaf(d[j][e] * wv[j][e], v[j][e], em);
          }
        }
        const float rstd = rsqrtf(fmaf(row_sum<LPR>(ss), inv_d, eps));
        const float mean = row_sum<LPR>(em) * rstd * inv_d;
        T* dx = dst + (tau * H + hd) * D;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float m = v[j][e] * rstd;
            dw[part][j][e] = fmaf(d[j][e], m, dw[part][j][e]);
            v[j][e] = rstd * (d[j][e] * wv[j][e] - m * mean);
          }
          row_store<T, VEC>(dx + k.c[j], k.nv[j], v[j]);
        }
      }
    }
  }
  if (!part_w) return;   // uniform: no weight gradients wanted
  float* out = part_w + (long)blockIdx.x * 2 * D;
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VEC; ++e) red[(row0 * LPR + lane) * VEC + e] = dw[part][j][e];
      __syncthreads();
      for (int i = threadIdx.x; i < LPR * VEC; i += QK_NT) {
        const int c = LPR * VEC * j + i;
        if (c >= D) continue;
        float s = 0.f;
        for (int q = 0; q < RPB; ++q) s += red[q * LPR * VEC + i];
        out[(long)part * D + c] = s;
      }
    }
}

// The weights' gradients from the blocks' rows, 64 threads a column.
constexpr int QD_C = 16, QD_R = 64;
__global__ __launch_bounds__(QD_C * QD_R) void qk_dw_kernel(const float* part, int rows, int D,
                                                            float* dqw, float* dkw) {
  __shared__ float red[QD_R][QD_C + 1];
  const int c = threadIdx.x % QD_C, r0 = threadIdx.x / QD_C, i = blockIdx.x * QD_C + c;
  float s = 0.f;
  if (i < 2 * D)
#pragma unroll 8
    for (int r = r0; r < rows; r += QD_R) s += part[(long)r * 2 * D + i];
  red[r0][c] = s;
  __syncthreads();
  for (int n = QD_R / 2; n > 0; n /= 2) {
    if (r0 < n) red[r0][c] += red[r0 + n][c];
    __syncthreads();
  }
  float* out = i < D ? dqw : dkw;
  if (r0 == 0 && i < 2 * D && out) out[i % D] = red[0][c];
}

// ---------------------------------------------------------------------------
// Rows that one wave's lanes hold whole in pieces of VEC > 1 elements (aligned heads of up to 64
// pieces: 512 columns in pieces of eight, 256 of four, 128 of two): the partner of a rotated piece comes from its lane, and the rows of the
// next batch are on their way while one is computed.
// ---------------------------------------------------------------------------
constexpr int QK_UB = 2;   // rows of a thread in a batch of the backward

template <typename T, int VEC>
struct Piece {
  static constexpr int W = VEC * sizeof(T) / 4;
  uint32_t w[W];
};

template <typename T, int VEC>
__device__ __forceinline__ void piece_load(Piece<T, VEC>& r, const T* p) {
  if constexpr (Piece<T, VEC>::W == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    r.w[0] = x.x, r.w[1] = x.y, r.w[2] = x.z, r.w[3] = x.w;
  } else if constexpr (Piece<T, VEC>::W == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    r.w[0] = x.x, r.w[1] = x.y;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void piece_values(const Piece<T, VEC>& r, float (&x)[VEC]) {
#pragma unroll
  for (int i = 0; i < Piece<T, VEC>::W; ++i) {
    if constexpr (sizeof(T) == 2) {
      x[2 * i] = bf16_lo(r.w[i]);
      x[2 * i + 1] = bf16_hi(r.w[i]);
    } else {
      x[i] = __uint_as_float(r.w[i]);
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void piece_of_lane(Piece<T, VEC>& r, int lane4) {
#pragma unroll
  for (int i = 0; i < Piece<T, VEC>::W; ++i)
    r.w[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(lane4, (int)r.w[i]);
}

// Element offsets of the block's tokens in q and k (and in their gradients).
__device__ __forceinline__ void token_offsets(const tops_gla_qk_args& a, long tau0, int nt,
                                              bool backward, long (*off)[4]) {
  const int k = threadIdx.x;
  if (k >= nt) return;
  const uint32_t tau = (uint32_t)(tau0 + k), bb = tau / (uint32_t)a.T;   // B T < 2^31
  const long b = bb, t = tau - bb * (uint32_t)a.T;
  off[k][0] = b * a.q_sb + t * a.q_st;
  off[k][1] = b * a.k_sb + t * a.k_st;
  if (backward) {
    off[k][2] = b * a.dq_sb + t * a.dq_st;
    off[k][3] = b * a.dk_sb + t * a.dk_st;
  }
}

// A lane's place in a row: its piece, the piece's partner, and what a rotation does with it.
template <int VEC, int LPR, bool INTER>
struct Lane {
  static constexpr bool EACH = VEC == 2 && !INTER;   // partners by the element, not the piece
  int c, f, lane4;
  bool in, rot, hi;
  int fe[2], pe[2], lane4e[2], odd;   // EACH: an element's frequency, partner's column and lane
  bool hie[2];
  __device__ __forceinline__ Lane(int D, int R) {
    const int lane = threadIdx.x % LPR, R2 = R / 2;
    c = lane * VEC;
    in = c < D;
    rot = c < R;
    hi = !INTER && rot && c >= R2;
    f = !rot ? 0 : INTER ? c / 2 : hi ? c - R2 : c;
    const int m = INTER || !rot ? 0 : hi ? -(R2 / VEC) : R2 / VEC;
    lane4 = 4 * ((threadIdx.x & 63) + m);
    if (EACH) {
      // half the rotated columns may be odd in number: the elements of a piece then have their
      // partners in two pieces, and one piece lies on both sides of the middle
      odd = R2 & 1;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        hie[e] = rot && c + e >= R2;
        fe[e] = !rot ? 0 : hie[e] ? c + e - R2 : c + e;
        pe[e] = !rot ? c + e : hie[e] ? c + e - R2 : c + e + R2;
        lane4e[e] = 4 * ((threadIdx.x & 63) + pe[e] / 2 - c / 2);
      }
    }
  }
  // whether an element is the second one of its pair, which the first is added to when it turns
  __device__ __forceinline__ bool second(int e) const { return EACH ? hie[e] : hi; }
  // column of the partner's piece
  __device__ __forceinline__ int pc(int R) const {
    return INTER || !rot ? c : hi ? c - R / 2 : c + R / 2;
  }
};

// The values of a piece's partners; BACK: those of second elements negated, as a turn back has them.
template <bool BACK, typename T, int VEC, int LPR, bool INTER>
__device__ __forceinline__ void partners(const Piece<T, VEC>& x, const Lane<VEC, LPR, INTER>& l,
                                         float (&p)[VEC]) {
  if constexpr (Lane<VEC, LPR, INTER>::EACH) {
    constexpr int W = Piece<T, VEC>::W;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      Piece<T, VEC> r;
      float v[VEC];
#pragma unroll
      for (int i = 0; i < W; ++i)
        r.w[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(l.lane4e[e], (int)x.w[i]);
      piece_values<T, VEC>(r, v);
      p[e] = l.odd ? v[1 - e] : v[e];
      if (BACK && l.hie[e]) p[e] = -p[e];
    }
  } else if constexpr (!INTER) {
    Piece<T, VEC> r = x;
    piece_of_lane<T, VEC>(r, l.lane4);
    if (BACK) {
      const uint32_t flip = l.hi ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
      for (int i = 0; i < Piece<T, VEC>::W; ++i) r.w[i] ^= flip;
    }
    piece_values<T, VEC>(r, p);
  }
}

// x turned by a token's angles cs, xp being its partners with their signs; whole pairs (INTER) turn
// by sign times the angles.
template <int VEC, int LPR, bool INTER>
__device__ __forceinline__ void turn_piece(float (&x)[VEC], const float (&xp)[VEC],
                                           const float2* cs, const Lane<VEC, LPR, INTER>& l, int R,
                                           float sign) {
  if constexpr (Lane<VEC, LPR, INTER>::EACH) {
    if (l.rot)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 k = cs[l.fe[e]];
        x[e] = fmaf(xp[e], k.y, x[e] * k.x);
      }
  } else if constexpr (INTER) {
    turn<VEC, INTER>(x, xp, cs + l.f, l.rot, l.hi, l.c, R, sign);
  } else if (l.rot) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float2 k = cs[l.f + e];
      x[e] = fmaf(xp[e], k.y, x[e] * k.x);
    }
  }
}

// `magic[p]` = ceil(2^32 / heads of part p): row / heads = mulhi(row, magic) for row < 2^16.
template <typename T, int VEC, int LPR, bool INTER, int QK_U>
__global__ __launch_bounds__(QK_NT) void qk_fwd_rows_kernel(tops_gla_qk_args a, int tb,
                                                            uint32_t magic_q, uint32_t magic_k) {
  extern __shared__ float2 cs[];
  __shared__ long off[QK_MAXTB][4];
  constexpr int RPB = QK_NT / LPR;
  constexpr bool PAIR = !INTER;
  const int row0 = threadIdx.x / LPR;
  const int D = (int)a.D, R = (int)a.R, R2 = R / 2;
  const long tokens = a.batch * a.T, tau0 = (long)blockIdx.x * tb;
  const int nt = (int)min((long)tb, tokens - tau0);
  const Lane<VEC, LPR, INTER> l(D, R);
  const int cl = l.in ? l.c : 0;
  token_offsets(a, tau0, nt, false, off);
  __syncthreads();
  const int rq = nt * (int)a.Hq, rk = nt * (int)a.Hk;   // rows of the two parts, and batches
  const int nbq = (rq + RPB * QK_U - 1) / (RPB * QK_U), nb = nbq + (rk + RPB * QK_U - 1) / (RPB * QK_U);
  Piece<T, VEC> nx[QK_U];
  auto load = [&](int i) {
    const bool part = i >= nbq;
    const int H = (int)(part ? a.Hk : a.Hq), rows = part ? rk : rq;
    const uint32_t magic = part ? magic_k : magic_q;
    const T* src = (const T*)(part ? a.k : a.q);
    const long sh = part ? a.k_sh : a.q_sh;
    const int r0 = (i - (part ? nbq : 0)) * RPB * QK_U + row0;
#pragma unroll
    for (int u = 0; u < QK_U; ++u) {
      const int r = min(r0 + u * RPB, rows - 1);
      const int tk = H == 1 ? r : (int)__umulhi((uint32_t)r, magic);
      piece_load<T, VEC>(nx[u], src + off[tk][part] + (r - tk * H) * sh + cl);
    }
  };
  float wv[VEC], wp[VEC];
  auto weights = [&](int part) {
    const float* w = part ? a.kw : a.qw;
    const int pc = l.in ? l.pc(R) : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      wv[e] = w ? w[cl + e] : 1.f;
      wp[e] = !w ? 1.f : Lane<VEC, LPR, INTER>::EACH ? w[l.in ? l.pe[e] : 0] : w[pc + e];
      if (PAIR && !l.second(e)) wp[e] = -wp[e];   // the sign of a pair's first half
    }
  };
  if (nb > 0) load(0);
  weights(nbq == 0);
  angles(a, tau0, nt, cs);
  __syncthreads();
  const float inv_d = 1.f / (float)D, eps = (float)a.eps;
#pragma unroll 1
  for (int i = 0; i < nb; ++i) {
    const bool part = i >= nbq;
    if (i == nbq && i > 0) weights(1);
    Piece<T, VEC> x[QK_U];
#pragma unroll
    for (int u = 0; u < QK_U; ++u) x[u] = nx[u];
    if (i + 1 < nb) load(i + 1);
    const int H = (int)(part ? a.Hk : a.Hq), rows = part ? rk : rq;
    const uint32_t magic = part ? magic_k : magic_q;
    T* dst = (T*)(part ? a.ko : a.qo) + tau0 * H * D;
    const int r0 = (i - (part ? nbq : 0)) * RPB * QK_U + row0;
#pragma unroll
    for (int u = 0; u < QK_U; ++u) {
      const int r = r0 + u * RPB;
      float v[VEC], p[VEC], ss = 0.f;
      piece_values<T, VEC>(x[u], v);
      if (PAIR) partners<false>(x[u], l, p);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss = fmaf(v[e], v[e], ss);
      const float rstd = rsqrtf(fmaf(row_sum<LPR>(l.in ? ss : 0.f), inv_d, eps));
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] *= wv[e];
        if (PAIR) p[e] *= wp[e];
      }
      if (r < rows && l.in) {
        const int tk = H == 1 ? r : (int)__umulhi((uint32_t)r, magic);
        turn_piece<VEC, LPR, INTER>(v, p, cs + tk * R2, l, R, 1.f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= rstd;
        store_run<T, VEC>(dst + (long)r * D + l.c, v);
      }
    }
  }
}

template <typename T, int VEC, int LPR, bool INTER>
__global__ __launch_bounds__(QK_NT) void qk_bwd_rows_kernel(tops_gla_qk_args a, long ngroups,
                                                            int tb, uint32_t magic_q,
                                                            uint32_t magic_k, float* part_w) {
  extern __shared__ float2 cs[];
  __shared__ float red[QK_NT * VEC];
  __shared__ long off[QK_MAXTB][4];
  constexpr int RPB = QK_NT / LPR;
  constexpr bool PAIR = !INTER;
  const int row0 = threadIdx.x / LPR;
  const int D = (int)a.D, R = (int)a.R, R2 = R / 2;
  const long tokens = a.batch * a.T;
  const Lane<VEC, LPR, INTER> l(D, R);
  const int cl = l.in ? l.c : 0;
  const float inv_d = 1.f / (float)D, eps = (float)a.eps;
  float dw[2][VEC] = {};
  for (long g = blockIdx.x; g < ngroups; g += gridDim.x) {
    const long tau0 = g * tb;
    const int nt = (int)min((long)tb, tokens - tau0);
    const int rq = nt * (int)a.Hq, rk = nt * (int)a.Hk;
    const int nbq = (rq + RPB * QK_UB - 1) / (RPB * QK_UB),
              nb = nbq + (rk + RPB * QK_UB - 1) / (RPB * QK_UB);
    __syncthreads();
    token_offsets(a, tau0, nt, true, off);
    __syncthreads();
    Piece<T, VEC> nx[QK_UB], ng[QK_UB];
    auto load = [&](int i) {
      const bool part = i >= nbq;
      const int H = (int)(part ? a.Hk : a.Hq), rows = part ? rk : rq;
      const uint32_t magic = part ? magic_k : magic_q;
      const T* src = (const T*)(part ? a.k : a.q);
      const T* gsrc = (const T*)(part ? a.dko : a.dqo);
      const long sh = part ? a.k_sh : a.q_sh, gh = part ? a.dk_sh : a.dq_sh;
      const int r0 = (i - (part ? nbq : 0)) * RPB * QK_UB + row0;
#pragma unroll
      for (int u = 0; u < QK_UB; ++u) {
        const int r = min(r0 + u * RPB, rows - 1);
        const int tk = H == 1 ? r : (int)__umulhi((uint32_t)r, magic), hd = r - tk * H;
        piece_load<T, VEC>(nx[u], src + off[tk][part] + hd * sh + cl);
        piece_load<T, VEC>(ng[u], gsrc + off[tk][2 + part] + hd * gh + cl);
      }
    };
    if (nb > 0) load(0);
    angles(a, tau0, nt, cs);
    __syncthreads();
    float wv[VEC];
#pragma unroll 1
    for (int i = 0; i < nb; ++i) {
      const bool part = i >= nbq;
      if (i == 0 || i == nbq) {
        const float* w = part ? a.kw : a.qw;
#pragma unroll
        for (int e = 0; e < VEC; ++e) wv[e] = w ? w[cl + e] : 1.f;
      }
      Piece<T, VEC> x[QK_UB], gy[QK_UB];
#pragma unroll
      for (int u = 0; u < QK_UB; ++u) x[u] = nx[u], gy[u] = ng[u];
      if (i + 1 < nb) load(i + 1);
      const int H = (int)(part ? a.Hk : a.Hq), rows = part ? rk : rq;
      const uint32_t magic = part ? magic_k : magic_q;
      T* dst = (T*)(part ? a.dk : a.dq) + tau0 * H * D;
      const int r0 = (i - (part ? nbq : 0)) * RPB * QK_UB + row0;
#pragma unroll
      for (int u = 0; u < QK_UB; ++u) {
        const int r = r0 + u * RPB;
        const bool on = r < rows && l.in;
        const int tk = H == 1 ? min(r, nt - 1)
                              : (int)__umulhi((uint32_t)min(r, rows - 1), magic);
        float v[VEC], d[VEC], p[VEC], ss = 0.f, em = 0.f;
        piece_values<T, VEC>(x[u], v);
        piece_values<T, VEC>(gy[u], d);
        if (PAIR) partners<true>(gy[u], l, p);
        turn_piece<VEC, LPR, INTER>(d, p, cs + tk * R2, l, R, -1.f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          ss = fmaf(v[e], v[e], ss);
          em = fmaf(d[e] * wv[e], v[e], em);
        }
        const float rstd = rsqrtf(fmaf(row_sum<LPR>(l.in ? ss : 0.f), inv_d, eps));
        const float mean = row_sum<LPR>(l.in ? em : 0.f) * rstd * inv_d;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float m = v[e] * rstd, t = on ? d[e] * m : 0.f;
          if (part)
            dw[1][e] += t;
          else
            dw[0][e] += t;
          v[e] = rstd * (d[e] * wv[e] - m * mean);
        }
        if (on) store_run<T, VEC>(dst + (long)r * D + l.c, v);
      }
    }
  }
  if (!part_w) return;   // uniform: no weight gradients wanted
  float* out = part_w + (long)blockIdx.x * 2 * D;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[threadIdx.x * VEC + e] = dw[part][e];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += QK_NT) {
      float s = 0.f;
      for (int q = 0; q < RPB; ++q) s += red[q * LPR * VEC + i];
      out[(long)part * D + i] = s;
    }
  }
}

constexpr long kQkBlocks = 1024;   // of the backward: rows of partial weight gradients

// Tokens of a block at a time, as long as the blocks fill the device: a block whose threads have
// several batches of rows pays less for its start (16 + 16 heads of 128 columns, 32768 tokens: 161 us
// forward with 4 tokens a block, 115 with 16; backward 174 with 4, 164 with 8).
int tokens_per_block(long tokens, long heads, bool backward) {
  int tb = 1;
  while (tb < QK_MAXTB && tb * heads < (backward ? 256 : 512) && tokens >= 2048L * tb) tb *= 2;
  return tb;
}
uint32_t magic_of(long heads) { return heads < 2 ? 0 : (uint32_t)(((1ULL << 32) + heads - 1) / heads); }

// A block's rows are at most 2^16 (heads are, and more tokens than one only for fewer than 512 of
// them), as a row's index times the magic number has to be exact.
template <typename T, int VEC, int LPR>
hipError_t qk_rows_launch(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  const long tokens = a.batch * a.T;
  const int tb = tokens_per_block(tokens, a.Hq + a.Hk, backward);
  const long groups = (tokens + tb - 1) / tb;
  const size_t lds = (size_t)tb * (a.R / 2) * sizeof(float2);
  const uint32_t mq = magic_of(a.Hq), mk = magic_of(a.Hk);
  const dim3 nt(QK_NT);
  if (!backward) {
    const dim3 grid((unsigned)groups);
    // four rows of a thread in a batch, one where a block has no more of them
    const bool few = tb * std::max(a.Hq, a.Hk) <= 2 * (QK_NT / LPR);
    if (a.interleaved && few)
      hipLaunchKernelGGL((qk_fwd_rows_kernel<T, VEC, LPR, true, 1>), grid, nt, lds, st, a, tb, mq, mk);
    else if (a.interleaved)
      hipLaunchKernelGGL((qk_fwd_rows_kernel<T, VEC, LPR, true, 4>), grid, nt, lds, st, a, tb, mq, mk);
    else if (few)
      hipLaunchKernelGGL((qk_fwd_rows_kernel<T, VEC, LPR, false, 1>), grid, nt, lds, st, a, tb, mq, mk);
    else
      hipLaunchKernelGGL((qk_fwd_rows_kernel<T, VEC, LPR, false, 4>), grid, nt, lds, st, a, tb, mq, mk);
    return hipGetLastError();
  }
  const long blocks = std::min(groups, kQkBlocks);
  float* part = a.dqw || a.dkw ? (float*)a.ws : nullptr;
  if (blocks > 0) {
    const dim3 grid((unsigned)blocks);
    if (a.interleaved)
      hipLaunchKernelGGL((qk_bwd_rows_kernel<T, VEC, LPR, true>), grid, nt, lds, st, a, groups, tb,
                         mq, mk, part);
    else
      hipLaunchKernelGGL((qk_bwd_rows_kernel<T, VEC, LPR, false>), grid, nt, lds, st, a, groups, tb,
                         mq, mk, part);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (!a.dqw && !a.dkw) return hipSuccess;
  hipLaunchKernelGGL(qk_dw_kernel, dim3((unsigned)((2 * a.D + QD_C - 1) / QD_C)),
                     dim3(QD_C * QD_R), 0, st, part, (int)blocks, (int)a.D, a.dqw, a.dkw);
  return hipGetLastError();
}

template <typename T, int VEC, int LPR, int NI>
hipError_t qk_launch(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  const long tokens = a.batch * a.T;
  const int tb = tokens_per_block(tokens, a.Hq + a.Hk, backward);
  const long groups = (tokens + tb - 1) / tb;
  const size_t lds = (size_t)tb * (a.R / 2) * sizeof(float2);
  if (!backward) {
    if (a.interleaved)
      hipLaunchKernelGGL((qk_fwd_kernel<T, VEC, LPR, NI, true>), dim3((unsigned)groups), dim3(QK_NT),
                         lds, st, a, tb);
    else
      hipLaunchKernelGGL((qk_fwd_kernel<T, VEC, LPR, NI, false>), dim3((unsigned)groups),
                         dim3(QK_NT), lds, st, a, tb);
    return hipGetLastError();
  }
  const long blocks = std::min(groups, kQkBlocks);
  float* part = a.dqw || a.dkw ? (float*)a.ws : nullptr;
  if (blocks > 0) {
    if (a.interleaved)
      hipLaunchKernelGGL((qk_bwd_kernel<T, VEC, LPR, NI, true>), dim3((unsigned)blocks), dim3(QK_NT),
                         lds, st, a, groups, tb, part);
    else
      hipLaunchKernelGGL((qk_bwd_kernel<T, VEC, LPR, NI, false>), dim3((unsigned)blocks),
                         dim3(QK_NT), lds, st, a, groups, tb, part);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (part || a.dqw || a.dkw) {
    hipLaunchKernelGGL(qk_dw_kernel, dim3((unsigned)((2 * a.D + QD_C - 1) / QD_C)),
                       dim3(QD_C * QD_R), 0, st, part, (int)blocks, (int)a.D, a.dqw, a.dkw);
    return hipGetLastError();
  }
  return hipSuccess;
}

// Whole, aligned pieces of n elements in every row, and partners on such pieces.
bool pieces_of(const tops_gla_qk_args& a, bool backward, int n) {
  const long by = n * (a.dtype == DT_BF16 ? 2 : 4);
  if (a.D % n || (!a.interleaved && n > 2 && (a.R / 2) % n)) return false;
  for (int64_t s : {a.q_sb, a.q_st, a.q_sh, a.k_sb, a.k_st, a.k_sh})
    if (s % n) return false;
  for (const void* p : {a.q, a.k, (const void*)a.qo, (const void*)a.ko})
    if ((uintptr_t)p % by) return false;
  if (!backward) return true;
  for (int64_t s : {a.dq_sb, a.dq_st, a.dq_sh, a.dk_sb, a.dk_st, a.dk_sh})
    if (s % n) return false;
  for (const void* p : {a.dqo, a.dko, (const void*)a.dq, (const void*)a.dk})
    if ((uintptr_t)p % by) return false;
  return true;
}

// Pieces of two elements, for heads of up to 128 columns: 4 or 8 bytes a lane.
template <typename T>
hipError_t qk_pairs(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  if (a.D <= 32) return qk_rows_launch<T, 2, 16>(a, backward, st);
  if (a.D <= 64) return qk_rows_launch<T, 2, 32>(a, backward, st);
  return qk_rows_launch<T, 2, 64>(a, backward, st);
}

// Heads of an odd size, rows that are not aligned, and wide heads that are no whole pieces of four:
// an element a lane.
template <typename T>
hipError_t qk_elements(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  if (a.D <= 8) return qk_launch<T, 1, 8, 1>(a, backward, st);
  if (a.D <= 16) return qk_launch<T, 1, 16, 1>(a, backward, st);
  if (a.D <= 32) return qk_launch<T, 1, 32, 1>(a, backward, st);
  if (a.D <= 64) return qk_launch<T, 1, 64, 1>(a, backward, st);
  if (a.D <= 128) return qk_launch<T, 1, 64, 2>(a, backward, st);
  return qk_launch<T, 1, 64, 8>(a, backward, st);
}

template <typename T, int VEC>
hipError_t qk_rows(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  const long pieces = a.D / VEC;
  if (pieces <= 8) return qk_rows_launch<T, VEC, 8>(a, backward, st);
  if (pieces <= 16) return qk_rows_launch<T, VEC, 16>(a, backward, st);
  if (pieces <= 32) return qk_rows_launch<T, VEC, 32>(a, backward, st);
  constexpr int NI = 512 / VEC / 64;   // rows of up to 512 elements
  if constexpr (NI > 1)
    if (pieces > 64) return qk_launch<T, VEC, 64, NI>(a, backward, st);
  return qk_rows_launch<T, VEC, 64>(a, backward, st);
}

}  // namespace

long qk_norm_rope_blocks(long tokens, long heads) {
  const long tb = tokens_per_block(tokens, heads, false);
  return (tokens + tb - 1) / tb;
}
long qk_norm_rope_part_rows(long tokens) { return std::min(tokens, kQkBlocks); }

hipError_t run_qk_norm_rope(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  if (a.batch * a.T == 0 && !backward) return hipSuccess;
  if (a.dtype == DT_BF16) {
    if (pieces_of(a, backward, 8)) return qk_rows<bf16, 8>(a, backward, st);
    if (pieces_of(a, backward, 4)) return qk_rows<bf16, 4>(a, backward, st);
    if (a.D <= 128 && pieces_of(a, backward, 2)) return qk_pairs<bf16>(a, backward, st);
    return qk_elements<bf16>(a, backward, st);
  }
  if (pieces_of(a, backward, 4)) return qk_rows<float, 4>(a, backward, st);
  if (a.D <= 128 && pieces_of(a, backward, 2)) return qk_pairs<float>(a, backward, st);
  return qk_elements<float>(a, backward, st);
}

}  // namespace tops
