// Norms of queries and keys for each head with the position rotation in the same pass, forward
// and backward (include/tops_gla_ssm.h).
//
// Bound by memory: a head's row is read and written once. LPR lanes hold a row, VEC elements
// each, so that its mean square is a sum over LPR lanes; the partner of a rotated element is
// read again (it is in the cache) instead of moved between lanes. cos and sin of a token's angles
// are formed once for all its heads, in LDS: the angle is taken in turns in 64 bits, where a far
// position times a frequency keeps its fraction, and only the fraction is rounded to 32.
#include "ssm.hpp"

namespace tops {

namespace {

constexpr int QK_NT = 256;
constexpr int QK_TB = 4;   // tokens whose angles a block forms at a time

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
    const long tau = tau0 + k, b = tau / a.T, t = tau - b * a.T;
    long pos = t;
    if (a.positions) {
      const long at = b * a.pos_sb + t;
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

// The weights' gradients from the blocks' rows, a wave a column.
__global__ __launch_bounds__(QK_NT) void qk_dw_kernel(const float* part, int rows, int D,
                                                      float* dqw, float* dkw) {
  const int i = blockIdx.x * (QK_NT / 64) + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (i >= 2 * D) return;
  float s = 0.f;
  for (int r = lane; r < rows; r += 64) s += part[(long)r * 2 * D + i];
  s = row_sum<64>(s);
  float* out = i < D ? dqw : dkw;
  if (lane == 0 && out) out[i % D] = s;
}

constexpr long kQkBlocks = 1024;   // of the backward: rows of partial weight gradients

// Tokens of a block: four where there are enough to fill the device.
int tokens_per_block(long tokens) { return tokens >= 4096 ? QK_TB : 1; }

template <typename T, int VEC, int LPR, int NI>
hipError_t qk_launch(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  const long tokens = a.batch * a.T;
  const int tb = tokens_per_block(tokens);
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
    hipLaunchKernelGGL(qk_dw_kernel, dim3((unsigned)((2 * a.D + 3) / 4)), dim3(QK_NT), 0, st, part,
                       (int)blocks, (int)a.D, a.dqw, a.dkw);
    return hipGetLastError();
  }
  return hipSuccess;
}

// Whole, aligned pieces of n elements in every row, and partners on such pieces.
bool pieces_of(const tops_gla_qk_args& a, bool backward, int n) {
  const long by = n * (a.dtype == DT_BF16 ? 2 : 4);
  if (a.D % n || (!a.interleaved && (a.R / 2) % n)) return false;
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

template <typename T, int VEC>
hipError_t qk_rows(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  const long pieces = (a.D + VEC - 1) / VEC;
  if (pieces <= 8) return qk_launch<T, VEC, 8, 1>(a, backward, st);
  if (pieces <= 16) return qk_launch<T, VEC, 16, 1>(a, backward, st);
  if (pieces <= 32) return qk_launch<T, VEC, 32, 1>(a, backward, st);
  constexpr int NI = 512 / VEC / 64;   // rows of up to 512 elements
  if constexpr (NI > 1)
    if (pieces <= 64) return qk_launch<T, VEC, 64, 1>(a, backward, st);
  return qk_launch<T, VEC, 64, NI>(a, backward, st);
}

}  // namespace

long qk_norm_rope_part_rows(long tokens) {
  const int tb = tokens_per_block(tokens);
  return std::min((tokens + tb - 1) / tb, kQkBlocks);
}

hipError_t run_qk_norm_rope(const tops_gla_qk_args& a, bool backward, hipStream_t st) {
  if (a.batch * a.T == 0 && !backward) return hipSuccess;
  if (a.dtype == DT_BF16) {
    if (pieces_of(a, backward, 8)) return qk_rows<bf16, 8>(a, backward, st);
    if (pieces_of(a, backward, 4)) return qk_rows<bf16, 4>(a, backward, st);
    return qk_rows<bf16, 1>(a, backward, st);
  }
  if (pieces_of(a, backward, 4)) return qk_rows<float, 4>(a, backward, st);
  return qk_rows<float, 1>(a, backward, st);
}

}  // namespace tops
