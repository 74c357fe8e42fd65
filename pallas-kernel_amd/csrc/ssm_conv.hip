// Causal depthwise convolution of width W <= 8 with the window carried in and out, forward and
// backward (include/tops_gla_ssm.h).
//
// Bound by memory. A thread walks a run of tokens for VEC channels (8 bytes a row) with the
// last W rows in registers, so that a row is loaded once by it, beside W - 1 rows at the run's
// ends; a block's threads lie along the channels. Packed sequences share one row of tokens: a
// run that holds a boundary is walked sequence by sequence. MI355X, B4 T8192 D4096 W4 bf16: forward
// 100 us (5.2 TB/s), backward 178 (x and dy in, dx out: 4.5 TB/s), the weights' sums 5.
#include "ssm.hpp"

namespace tops {

namespace {

constexpr int CV_NT = 256;
constexpr int CV_CX = 64;    // threads along the channels
constexpr int CV_U = 4;      // rows in flight, forward (8192 tokens, 2048 channels: 17.9 us, with 8 19.3)
constexpr int CV_UB = 8;     // and backward (32768 tokens, 4096 channels: 178 us, with 4 182)

// VEC consecutive elements of a row, at any address of theirs: the wide loads and stores need no
// alignment beyond the element's.
template <typename T, int VEC>
struct Row {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Row<T, VEC>& r, float (&x)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = to_f32(r.v[e]);
}
template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const float (&x)[VEC]) {
  Row<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = from_f32<T>(x[e]);
  *reinterpret_cast<Row<T, VEC>*>(p) = r;
}
template <typename T, int VEC>
__device__ __forceinline__ Row<T, VEC> get(const T* p) {
  return *reinterpret_cast<const Row<T, VEC>*>(p);
}

// First channel of the i-th thread along them, -1 past the last. Where D is no multiple of VEC the
// last thread takes the last VEC channels: some of them twice, to the same values.
template <int VEC>
__device__ __forceinline__ int channel_of(const tops_gla_conv_args& a, int i) {
  const int c = i * VEC, D = (int)a.D;
  return c >= D ? -1 : min(c, D - VEC);
}

// First and end token of sequence s, in the flattened tokens.
__device__ __forceinline__ void conv_seq(const tops_gla_conv_args& a, int s, long& bos, long& eos) {
  if (a.cu) {
    bos = a.cu[s];
    eos = a.cu[s + 1];
  } else {
    bos = s * a.T;
    eos = bos + a.T;
  }
}
// The sequence of a flattened token.
__device__ __forceinline__ int conv_find(const tops_gla_conv_args& a, long tau) {
  if (!a.cu) return (int)(tau / a.T);
  int lo = 0, hi = (int)a.nseq - 1;   // the last one that starts at or before the token
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (a.cu[m] <= tau) lo = m; else hi = m - 1;
  }
  return lo;
}
// Pointer to input row `r` tokens after the sequence's start (r >= 0).
template <typename T>
__device__ __forceinline__ const T* in_row(const void* base, long sb, long st,
                                           const tops_gla_conv_args& a, int s, long bos, long r) {
  return (const T*)base + (a.cu ? (bos + r) * st : s * sb + r * st);
}

// The W - 1 rows before token r of sequence s, oldest first, into win[1 ..].
template <typename T, int VEC, int W>
__device__ __forceinline__ void head(const tops_gla_conv_args& a, int s, long bos, long r, int c,
                                     float (&win)[W][VEC]) {
#pragma unroll
  for (int j = 1; j < W; ++j) {
    const long p = r - W + j;
#pragma unroll
    for (int e = 0; e < VEC; ++e) win[j][e] = 0.f;
    if (p >= 0)
      unpack<T, VEC>(get<T, VEC>(in_row<T>(a.x, a.x_sb, a.x_st, a, s, bos, p) + c), win[j]);
    else if (a.init)
      unpack<T, VEC>(get<T, VEC>((const T*)a.init + ((long)s * W + W + p) * a.D + c), win[j]);
  }
}

template <typename TW, int VEC, int W>
__device__ __forceinline__ void weights_of(const TW* w0, const TW* b0, int c, float (&w)[W][VEC],
                                           float (&b)[VEC]) {
  float x[VEC * W];
  const TW* p = w0 + (long)c * W;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float v[VEC];
    unpack<TW, VEC>(get<TW, VEC>(p + VEC * j), v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[VEC * j + e] = v[e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    b[e] = b0 ? to_f32(b0[c + e]) : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = x[e * W + j];
  }
}
template <int VEC, int W>
__device__ __forceinline__ void weights(const tops_gla_conv_args& a, int c, float (&w)[W][VEC],
                                        float (&b)[VEC]) {
  if (a.w_dtype == DT_BF16)
    weights_of<bf16, VEC, W>((const bf16*)a.w, (const bf16*)a.bias, c, w, b);
  else
    weights_of<float, VEC, W>((const float*)a.w, (const float*)a.bias, c, w, b);
}

template <int VEC, int W>
__device__ __forceinline__ void push(float (&win)[W][VEC], const float (&x)[VEC]) {
#pragma unroll
  for (int j = 0; j + 1 < W; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) win[j][e] = win[j + 1][e];
#pragma unroll
  for (int e = 0; e < VEC; ++e) win[W - 1][e] = x[e];
}

template <int VEC, int W>
__device__ __forceinline__ void conv_of(const float (&win)[W][VEC], const float (&w)[W][VEC],
                                        const float (&b)[VEC], float (&z)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    z[e] = b[e];
#pragma unroll
    for (int j = 0; j < W; ++j) z[e] = fmaf(w[j][e], win[j][e], z[e]);
  }
}

// Row r of the final state of sequence s (its last W inputs, those before the first token from
// the initial state).
template <typename T, int VEC>
__device__ __forceinline__ void final_row(const tops_gla_conv_args& a, int s, int r, int c) {
  long bos, eos;
  conv_seq(a, s, bos, eos);
  const int W = (int)a.W;
  const long p = eos - bos - W + r;
  Row<T, VEC> x;
#pragma unroll
  for (int e = 0; e < VEC; ++e) x.v[e] = from_f32<T>(0.f);
  if (p >= 0)
    x = get<T, VEC>(in_row<T>(a.x, a.x_sb, a.x_st, a, s, bos, p) + c);
  else if (a.init)
    x = get<T, VEC>((const T*)a.init + ((long)s * W + W + p) * a.D + c);
  *reinterpret_cast<Row<T, VEC>*>((T*)a.final_state + ((long)s * W + r) * a.D + c) = x;
}

// Blocks: `slabs` channel slabs of each group of 4 runs of `run` tokens, then of the final
// states' rows.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(CV_NT) void conv_fwd_kernel(tops_gla_conv_args a, int run, long tiles,
                                                         int slabs) {
  const int slab = blockIdx.x % slabs;
  const long group = blockIdx.x / slabs;
  const int c = channel_of<VEC>(a, slab * CV_CX + threadIdx.x % CV_CX);
  if (c < 0) return;
  const int ry = __builtin_amdgcn_readfirstlane(threadIdx.x / CV_CX);
  if (group >= tiles) {
    const long i = (group - tiles) * 4 + ry;
    if (i < a.nseq * W) final_row<T, VEC>(a, (int)(i / W), (int)(i % W), c);
    return;
  }
  const long tokens = a.batch * a.T;
  long tau = (group * 4 + ry) * run;
  const long end = min(tokens, tau + run);
  if (tau >= end) return;
  float w[W][VEC], b[VEC], win[W][VEC];
  weights<VEC, W>(a, c, w, b);
  for (int s = conv_find(a, tau); tau < end && s < a.nseq; ++s) {
    long bos, eos;
    conv_seq(a, s, bos, eos);
    const long hi = min(end, eos);
    if (tau >= hi) continue;   // an empty sequence
    head<T, VEC, W>(a, s, bos, tau - bos, c, win);
    const T* x = in_row<T>(a.x, a.x_sb, a.x_st, a, s, bos, tau - bos) + c;
    T* y = (T*)a.y + tau * a.D + c;
    for (long n = hi - tau; n > 0; n -= CV_U, x += CV_U * a.x_st, y += CV_U * a.D) {
      Row<T, VEC> r[CV_U];
#pragma unroll
      for (int i = 0; i < CV_U; ++i) r[i] = get<T, VEC>(x + (i < n ? i : 0) * a.x_st);
#pragma unroll
      for (int i = 0; i < CV_U; ++i) {
        float v[VEC], z[VEC];
        unpack<T, VEC>(r[i], v);
        push<VEC, W>(win, v);
        conv_of<VEC, W>(win, w, b, z);
        if (a.silu)
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[e] *= sigmoid(z[e]);
        if (i < n) put<T, VEC>(y + i * a.D, z);
      }
    }
    tau = hi;
  }
}

// dz_t = dy_t act'(z_t); dx_t = sum_m w[W - 1 - m] dz_{t + m}; dw[j] = sum_t dz_t x_{t - W + 1 + j}.
// A run recomputes the z of the W - 1 tokens after it, whose dz its inputs reach.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(CV_NT) void conv_bwd_kernel(tops_gla_conv_args a, int run,
                                                         int slabs, float* part) {
  __shared__ float red[3][CV_CX][VEC + 1];
  const int cx = threadIdx.x % CV_CX;
  const int ry = __builtin_amdgcn_readfirstlane(threadIdx.x / CV_CX);
  const int slab = blockIdx.x % slabs;
  const long group = blockIdx.x / slabs;
  const int c = channel_of<VEC>(a, slab * CV_CX + cx);
  const bool live = c >= 0;
  const long tokens = a.batch * a.T;
  long tau = (group * 4 + ry) * run;
  const long end = min(tokens, tau + run);
  float dw[W + 1][VEC] = {};
  if (live && tau < end) {
    float w[W][VEC], b[VEC], win[W][VEC], dz[W][VEC];
    weights<VEC, W>(a, c, w, b);
    for (int s = conv_find(a, tau); tau < end && s < a.nseq; ++s) {
      long bos, eos;
      conv_seq(a, s, bos, eos);
      const long hi = min(end, eos);
      if (tau >= hi) continue;
      head<T, VEC, W>(a, s, bos, tau - bos, c, win);
#pragma unroll
      for (int j = 0; j < W; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) dz[j][e] = 0.f;
      // token t = tau + n: its dz, then the gradient of input t - W + 1
      const long last = hi - tau + W - 1;          // tokens walked, W - 1 past the run
      const long have = min(last, eos - tau);      // those of the sequence
      const T* x = in_row<T>(a.x, a.x_sb, a.x_st, a, s, bos, tau - bos) + c;
      const T* g = in_row<T>(a.dy, a.dy_sb, a.dy_st, a, s, bos, tau - bos) + c;
      for (long n = 0; n < last; n += CV_UB) {
        Row<T, VEC> xr[CV_UB], gr[CV_UB];
#pragma unroll
        for (int i = 0; i < CV_UB; ++i) {
          const long k = min(n + i, have - 1);
          xr[i] = get<T, VEC>(x + k * a.x_st);
          gr[i] = get<T, VEC>(g + k * a.dy_st);
        }
#pragma unroll
        for (int i = 0; i < CV_UB; ++i) {
          const long k = n + i;
          float v[VEC], z[VEC], d[VEC];
          unpack<T, VEC>(xr[i], v);
          unpack<T, VEC>(gr[i], d);
          push<VEC, W>(win, v);
          if (a.silu) {
            conv_of<VEC, W>(win, w, b, z);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float sg = sigmoid(z[e]);
              d[e] *= sg * fmaf(z[e], 1.f - sg, 1.f);
            }
          }
          if (k >= have)
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = 0.f;
          push<VEC, W>(dz, d);
          if (k < hi - tau)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
#pragma unroll
              for (int j = 0; j < W; ++j) dw[j][e] = fmaf(d[e], win[j][e], dw[j][e]);
              dw[W][e] += d[e];
            }
          const long t = tau + k - (W - 1);
          if (k >= W - 1 && t < hi) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              o[e] = 0.f;
#pragma unroll
              for (int m = 0; m < W; ++m) o[e] = fmaf(w[W - 1 - m][e], dz[m][e], o[e]);
            }
            if (a.dfinal && t >= eos - W) {
              float f[VEC];
              unpack<T, VEC>(get<T, VEC>((const T*)a.dfinal +
                                         ((long)s * W + (t - (eos - W))) * a.D + c), f);
#pragma unroll
              for (int e = 0; e < VEC; ++e) o[e] += f[e];
            }
            put<T, VEC>((T*)a.dx + t * a.D + c, o);
          }
        }
      }
      tau = hi;
    }
  }
  if (!part) return;   // uniform: no weight gradients wanted
  float* row = part + group * (W + 1) * a.D;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    if (ry > 0)
#pragma unroll
      for (int e = 0; e < VEC; ++e) red[ry - 1][cx][e] = dw[j][e];
    __syncthreads();
    if (ry == 0 && live)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float t = (dw[j][e] + red[0][cx][e]) + (red[1][cx][e] + red[2][cx][e]);
        if (j < W)
          row[(long)(c + e) * W + j] = t;
        else
          row[(long)W * a.D + c + e] = t;
      }
    __syncthreads();
  }
}

// Gradient of the initial states: row i holds input i - W of its sequence.
template <typename T, int W>
__global__ __launch_bounds__(CV_NT) void conv_dinit_kernel(tops_gla_conv_args a, int slabs) {
  const int c = blockIdx.x % slabs * CV_NT + threadIdx.x, s = blockIdx.x / slabs;
  if (c >= a.D) return;
  long bos, eos;
  conv_seq(a, s, bos, eos);
  const long len = eos - bos;
  float w[W][1], b[1], win[W][1], dz[W];
  weights<1, W>(a, c, w, b);
  head<T, 1, W>(a, s, bos, 0, c, win);
#pragma unroll
  for (int k = 0; k < W; ++k) {   // dz of the first W - 1 tokens
    dz[k] = 0.f;
    if (k < W - 1 && k < len) {
      float v[1], z[1];
      v[0] = to_f32(in_row<T>(a.x, a.x_sb, a.x_st, a, s, bos, k)[c]);
      push<1, W>(win, v);
      conv_of<1, W>(win, w, b, z);
      float d = to_f32(in_row<T>(a.dy, a.dy_sb, a.dy_st, a, s, bos, k)[c]);
      if (a.silu) {
        const float sg = sigmoid(z[0]);
        d *= sg * fmaf(z[0], 1.f - sg, 1.f);
      }
      dz[k] = d;
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {   // input i - W in the window of token k at i - 1 - k
      const int j = i - 1 - k;
      if (j >= 0) o = fmaf(w[j][0], dz[k], o);
    }
    if (a.dfinal && i - len >= 0)   // kept as row i - len of the final state
      o += to_f32(((const T*)a.dfinal)[((long)s * W + (i - len)) * a.D + c]);
    ((T*)a.dinit)[((long)s * W + i) * a.D + c] = from_f32<T>(o);
  }
}

// The summed rows [D][W], [D] to the two outputs, 8 threads a column.
__global__ __launch_bounds__(256) void conv_dw_kernel(const float* __restrict__ part, int rows,
                                                      long m, long dw_n, void* dw, void* db,
                                                      int bf) {
  __shared__ float red[8][32];
  const int c = threadIdx.x % 32, row = threadIdx.x / 32;
  const long i = blockIdx.x * 32L + c;
  float s = 0.f;
  if (i < m)
#pragma unroll 8
    for (int r = row; r < rows; r += 8) s += part[r * m + i];
  red[row][c] = s;
  __syncthreads();
  if (row || i >= m) return;
  s = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) s += red[r][c];
  void* out = i < dw_n ? dw : db;
  const long at = i < dw_n ? i : i - dw_n;
  if (out && bf)
    ((bf16*)out)[at] = from_f32<bf16>(s);
  else if (out)
    ((float*)out)[at] = s;
}

// Tokens of a run: long ones re-read fewer rows at their ends, as long as the blocks (of 4 runs
// and 256 channels) fill the card.
int run_of(long tokens, long D) {
  int run = 128;
  while (run > 8 && (D + 255) / 256 * (tokens / (4 * run)) < 1024) run /= 2;
  return run;
}

template <typename T, int VEC, int W>
hipError_t conv_launch(const tops_gla_conv_args& a, bool backward, hipStream_t st) {
  const long tokens = a.batch * a.T;
  const int run = run_of(tokens, a.D);
  const long tiles = (tokens + 4L * run - 1) / (4L * run);
  const unsigned gx = (unsigned)((a.D + CV_CX * VEC - 1) / (CV_CX * VEC));
  if (!backward) {
    const long fin = a.final_state ? (a.nseq * W + 3) / 4 : 0;
    if (tiles + fin == 0) return hipSuccess;
    hipLaunchKernelGGL((conv_fwd_kernel<T, VEC, W>), dim3((unsigned)(gx * (tiles + fin))),
                       dim3(CV_NT), 0, st, a, run, tiles, (int)gx);
    return hipGetLastError();
  }
  if (tiles > 0) {
    hipLaunchKernelGGL((conv_bwd_kernel<T, VEC, W>), dim3((unsigned)(gx * tiles)), dim3(CV_NT), 0,
                       st, a, run, (int)gx, a.dw ? (float*)a.ws : nullptr);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (a.dw) {
    const long m = (W + 1) * a.D;
    hipLaunchKernelGGL(conv_dw_kernel, dim3((unsigned)((m + 31) / 32)), dim3(256), 0, st,
                       (const float*)a.ws, (int)tiles, m, W * a.D, a.dw, a.dbias,
                       (int)(a.w_dtype == DT_BF16));
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (a.dinit && a.nseq > 0) {
    const int ds = (int)((a.D + CV_NT - 1) / CV_NT);
    hipLaunchKernelGGL((conv_dinit_kernel<T, W>), dim3((unsigned)(ds * a.nseq)), dim3(CV_NT), 0, st,
                       a, ds);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <typename T, int W>
hipError_t conv_width(const tops_gla_conv_args& a, bool backward, hipStream_t st) {
  // 8 bytes of a row a thread: the backward holds 4 W + 2 rows in registers (with 16 bytes 256 of
  // them, one wave a SIMD: 249 us against 178 for 32768 tokens of 4096 channels, bf16), and the
  // forward of few tokens has more waves (8192 tokens, 2048 channels: 27 and 20 us)
  constexpr int VEC = 8 / (int)sizeof(T);
  if (a.D >= VEC) return conv_launch<T, VEC, W>(a, backward, st);
  return conv_launch<T, 1, W>(a, backward, st);
}

template <typename T>
hipError_t conv_any(const tops_gla_conv_args& a, bool backward, hipStream_t st) {
  switch (a.W) {
    case 1: return conv_width<T, 1>(a, backward, st);
    case 2: return conv_width<T, 2>(a, backward, st);
    case 3: return conv_width<T, 3>(a, backward, st);
    case 4: return conv_width<T, 4>(a, backward, st);
    case 5: return conv_width<T, 5>(a, backward, st);
    case 6: return conv_width<T, 6>(a, backward, st);
    case 7: return conv_width<T, 7>(a, backward, st);
    default: return conv_width<T, 8>(a, backward, st);
  }
}

hipError_t conv_run(const tops_gla_conv_args& a, bool backward, hipStream_t st) {
  if (a.D == 0) return hipSuccess;
  return a.dtype == DT_BF16 ? conv_any<bf16>(a, backward, st) : conv_any<float>(a, backward, st);
}

}  // namespace

long causal_conv_part_rows(long tokens, long D) {
  const long per = 4L * run_of(tokens, D);
  return (tokens + per - 1) / per;
}

hipError_t run_causal_conv_fwd(const tops_gla_conv_args& a, hipStream_t st) {
  return conv_run(a, false, st);
}
hipError_t run_causal_conv_bwd(const tops_gla_conv_args& a, hipStream_t st) {
  return conv_run(a, true, st);
}

}  // namespace tops
