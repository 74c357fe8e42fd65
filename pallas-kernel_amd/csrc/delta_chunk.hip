// The gated delta rule over chunks of C tokens, forward (include/tops_gla_delta.h).
//
// Within a chunk with the state S before it, G_i the sum of the log decays up to token i and
// D_ij = e^{G_i - G_j} for j <= i, the written values solve a unit triangular system:
//   (1 + A) N = beta (V - e^G (K S)),  A_ij = beta_i (k_i . k_j) D_ij below the diagonal.
// With Tm = (1 + A)^-1, which needs no state:
//   N = Tm (beta (V - e^G (K S))),   S <- e^{G_C} S + K^T (e^{G_C - G} N),
//   o = scale (e^G (Q S) + ((Q K^T) D) N).
// Here: Tm of every chunk at once. The states go from chunk to chunk, and the outputs with them
// (delta_scan.hip).
#include "delta.hpp"

namespace tops {

namespace {

// ---------------------------------------------------------------------------
// Tm and the vectors of a chunk
// ---------------------------------------------------------------------------

// X . Y over 16 with float operands: X row-major in LDS, Y in accumulator layout.
__device__ __forceinline__ void mma16(f32x4& acc, const float* X, int px, const f32x4& y,
                                      int lane) {
  const float4 x = *reinterpret_cast<const float4*>(X + (lane & 15) * px + 4 * (lane >> 4));
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y[2], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y[3], acc, 0, 0, 0);
}

// A block has a chunk and a key head, and goes through its value heads. K K^T on the matrix units;
// the inverse in float32: the 16 x 16 diagonal blocks by substitution, a lane a column, then the
// blocks below them, one diagonal after another: T_ij = -T_ii sum_k A_ik T_kj. Bound by the latency
// of these few steps: four blocks a CU, T where the keys were, gates on their way early: 16384 tokens
// of 16 heads of 128 keys in 53 us; the keys read and T written alone, 164 MB, would take 33.
template <typename T, int KP>
__global__ __launch_bounds__(256, 4) void delta_prep_kernel(DeltaParams p) {
  constexpr int C = delta_c<T>(), NB = C / 16, PK = pitch_of<T>(KP), PA = C + 4;
  // the keys, and then, for each value head, T
  constexpr int FIRST = std::max(C * PK * (int)sizeof(T), C * PA * 4);
  __shared__ __attribute__((aligned(16))) unsigned char first[FIRST];
  __shared__ __attribute__((aligned(16))) float sA[C * PA];
  T* sK = (T*)first;
  float* sT = (float*)first;
  __shared__ double sG[C];
  __shared__ float sBeta[C], sRk[C], sKK[C];
  __shared__ int sFirst;
  const tops_gla_delta_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int H = (int)a.H, HV = (int)a.HV, K = (int)a.K;
  const int chunk = (int)(blockIdx.x / H), h = (int)(blockIdx.x % H);
  const ChunkAt at = delta_chunk_at(a, C, chunk);
  // the first value head's gates on their way with the keys, the next one's while a head is worked on
  const long g_at = at.b * a.g_sb + (long)(at.t + min(lane, at.len - 1)) * a.g_st;
  const long b_at = at.b * a.beta_sb + (long)(at.t + min(lane, at.len - 1)) * a.beta_st;
  float g_next = 0.f, beta_next = 0.f;
  auto gates = [&](int hv) {
    if (wave == 0) {
      g_next = get_any(a.g, (int)a.g_dtype, g_at + hv);
      beta_next = get_any(a.beta, (int)a.beta_dtype, b_at + hv);
    }
  };
  gates(h * (HV / H));
  {
    TileFetch<T, C, KP, 256> f;
    f.get((const T*)a.k + at.b * a.k_sb + at.t * a.k_st + h * a.k_sh, a.k_st, at.len, K, tid);
    f.put(sK, PK, at.len, K, tid);
  }
  __syncthreads();
  {   // 1 / |k|: 256 / C threads a row
    constexpr int TR = 256 / C;
    const int row = tid / TR;
    float s = 0.f;
    if (a.l2norm) {
      for (int c = tid % TR; c < K; c += TR) {
        const float x = to_f32(sK[row * PK + c]);
        s = fmaf(x, x, s);
      }
    }
#pragma unroll
    for (int o = 1; o < TR; o <<= 1) s += __shfl_xor(s, o);
    if (tid % TR == 0) sRk[row] = a.l2norm ? rsqrtf(s + DELTA_L2_EPS) : 1.f;
  }
  f32x4 kk[NB];
  if (wave < NB) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      kk[j] = zero4();
      if (j <= wave) mma_tile<T>(kk[j], sK + wave * 16 * PK, PK, sK + j * 16 * PK, PK, KP, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r)   // the diagonal
        if (j == wave && (lane & 15) == 4 * (lane >> 4) + r) sKK[16 * j + (lane & 15)] = kk[j][r];
    }
  }
  __syncthreads();
  const int group = HV / H;
  for (int gi = 0; gi < group; ++gi) {
    const int hv = h * group + gi;
    const long unit = (long)chunk * HV + hv;
    if (wave == 0) {
      // From the first token on whose k, g or beta is not finite, the chunk has no tokens here: what
      // comes before it stays as it is, and what is made of the rest is set to NaN below.
      const bool bad = lane < at.len && !(fabsf(sKK[lane]) < INFINITY && g_next < INFINITY &&
                                          fabsf(beta_next) < INFINITY);
      const uint64_t any = __ballot(bad);
      const int first = any ? __ffsll((unsigned long long)any) - 1 : C;
      if (lane == 0) sFirst = first;
      const float g = lane < min(at.len, first) ? log_decay(g_next) : 0.f;
      const float beta = lane < min(at.len, first) ? beta_next : 0.f;
      double s = g;
#pragma unroll
      for (int o = 1; o < C; o <<= 1) {
        const double x = __shfl_up(s, o);
        if (lane >= o) s += x;
      }
      if (lane < C) {
        sG[lane] = s;
        sBeta[lane] = beta;
      }
    }
    if (gi + 1 < group) gates(hv + 1);
#pragma unroll
    for (int b = 0; b < C / 32; ++b)   // what is stored of T above the diagonal blocks
      sT[(32 * b + tid / 16) * PA + 32 * b + 16 + tid % 16] = 0.f;
    __syncthreads();
    const int first = sFirst;
    if (tid < C) {
      float* vec = delta_vec(p, unit);
      const double G = sG[tid];
      const bool in = tid < first;
      const float rk = in ? sRk[tid] : 0.f, e = in ? expf((float)G) : NAN;
      const float l = first < C ? NAN : expf((float)(sG[C - 1] - G));   // the state after the chunk
      if (tid == 0) delta_first(p, unit)[0] = first;
      vec[tid] = in ? e * rk : 0.f;
      vec[C + tid] = l * rk;
      vec[2 * C + tid] = sBeta[tid];
      vec[3 * C + tid] = rk;
      vec[4 * C + tid] = e;
      vec[5 * C + tid] = l;
      delta_gsum(p, unit)[tid] = G;
    }
    if (wave < NB) {
      const int row0 = 16 * wave + 4 * (lane >> 4);
      float f[4];
      double gr[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f[r] = sBeta[row0 + r] * sRk[row0 + r];
        gr[r] = sG[row0 + r];
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j > wave) continue;
        const int col = 16 * j + (lane & 15);
        const double gj = sG[col];
        const float rj = sRk[col];
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) d[r] = pinned(f[r] * rj * expf((float)(gr[r] - gj)));
#pragma unroll
        for (int r = 0; r < 4; ++r)   // a choice, no product: what is masked may be anything
          sA[(row0 + r) * PA + col] = row0 + r > col && row0 + r < first ? kk[j][r] * d[r] : 0.f;
      }
    }
    __syncthreads();
    if (wave < NB && lane < 16) {
      float x[16];
      const float* A = sA + 16 * wave * PA + 16 * wave;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == lane ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = fmaf(-A[i * PA + j], x[j], s);
        x[i] = s;
        sT[(16 * wave + i) * PA + 16 * wave + lane] = s;
      }
    }
#pragma unroll
    for (int d = 1; d < NB; ++d) {
      __syncthreads();
      if (wave < NB - d) {   // block (wave + d, wave)
        const int bi = wave + d, bj = wave;
        f32x4 m = zero4(), t = zero4();
#pragma unroll
        for (int k = 0; k < d; ++k) {   // A_ik T_kj, k from bj on
          const float* y = sT + (16 * (bj + k) + 4 * (lane >> 4)) * PA + 16 * bj + (lane & 15);
          const f32x4 yv = {y[0], y[PA], y[2 * PA], y[3 * PA]};
          mma16(m, sA + 16 * bi * PA + 16 * (bj + k), PA, yv, lane);
        }
        mma16(t, sT + 16 * bi * PA + 16 * bi, PA, m, lane);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sT[(16 * bi + 4 * (lane >> 4) + r) * PA + 16 * bj + (lane & 15)] = -t[r];
      }
    }
    __syncthreads();
    T* out = (T*)(p.Tm + unit * p.tri_bytes);
    constexpr int TRI = delta_blocks<T>() * 1024;
    for (int i = tid; i < TRI / 8; i += 256) {   // 8 elements of block x
      const int x = i / 128, row = i % 128 / 4, col = i % 4 * 8;
      const float* t = sT + (32 * (x > 0) + row) * PA + 32 * (x == 2) + col;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = t[e];
      const Whole<T> s = split_of<T, WHOLE<T>>(y);
#pragma unroll
      for (int part = 0; part < WHOLE<T>; ++part) st_frag(out + part * TRI + 8 * i, s.p[part]);
    }
    __syncthreads();
  }
}

long up(long n) { return (n + 255) / 256 * 256; }

}  // namespace

DeltaParams delta_layout(const tops_gla_delta_sizes& z, void* keep, void* ws) {
  DeltaParams p{};
  const long units = z.chunks * z.HV, segs = z.nsegs * z.HV;
  p.C = delta_chunk_of((int)z.dtype);
  p.KP = delta_key_pad(z.K);
  p.vec_bytes = 36 * p.C + 16;
  // bytes of an element in three parts and in two
  const long whole = z.dtype == DT_BF16 ? 2 * WHOLE<bf16> : 4, two = 4;
  p.tri_bytes = (z.dtype == DT_BF16 ? 3 : 1) * 1024 * whole;
  p.map_bytes = (long)p.KP * p.KP * whole;
  p.multi = z.nsegs > z.nseq;
  long at = 0;
  auto take = [&](void* base, long bytes) {
    char* x = (char*)base + at;
    at += up(bytes);
    return x;
  };
  const long ends = p.multi ? segs * z.K * z.V * 4 : 0, maps = p.multi ? segs * p.map_bytes : 0;
  p.vec = take(keep, units * p.vec_bytes);
  p.Tm = take(keep, units * p.tri_bytes);
  p.P = take(keep, z.train ? units * p.tri_bytes : 0);
  p.N = take(keep, z.train ? units * z.V * p.C * two : 0);
  p.S = take(keep, z.train ? units * z.V * p.KP * two : 0);
  p.E = (float*)take(keep, ends);
  p.M = take(keep, maps);
  p.Mt = take(keep, z.train ? maps : 0);
  p.keep_bytes = at;
  at = 0;
  p.dS = take(ws, units * z.V * p.KP * two);
  p.Y = take(ws, units * z.V * p.C * two);
  p.dE = (float*)take(ws, ends);
  p.ws_bytes = at;
  return p;
}

template <typename T, int KP>
static hipError_t prep(const DeltaParams& p, hipStream_t st) {
  delta_prep_kernel<T, KP><<<(unsigned)(p.a.chunks * p.a.H), 256, 0, st>>>(p);
  return hipGetLastError();
}
hipError_t run_delta_prep(const DeltaParams& p, hipStream_t st) {
  if (p.a.dtype == DT_BF16)
    return p.KP == 64 ? prep<bf16, 64>(p, st) : p.KP == 128 ? prep<bf16, 128>(p, st)
                                                            : prep<bf16, 256>(p, st);
  return p.KP == 64 ? prep<float, 64>(p, st) : p.KP == 128 ? prep<float, 128>(p, st)
                                                           : prep<float, 256>(p, st);
}

}  // namespace tops
