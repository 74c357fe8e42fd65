// The single-token forms: one step of the selective scan and of its convolution for each row of
// a serving batch, the states updated in place (include/tops_gla_ssm.h).
//
// Both are bound by the states' traffic (a row's state is read and written once), and for a few
// rows by the launch.
#include "ssm.hpp"

namespace tops {

namespace {

__device__ __forceinline__ long slot_of(const void* idx, bool idx64, int b) {
  if (!idx) return b;
  return idx64 ? (long)((const int64_t*)idx)[b] : (long)((const int32_t*)idx)[b];
}

// Sum over LPR adjacent lanes (a power of two up to 16).
template <int LPR>
__device__ __forceinline__ float sum_adjacent(float x) {
  if constexpr (LPR >= 2) x += dpp<0xb1>(x);
  if constexpr (LPR >= 4) x += dpp<0x4e>(x);
  if constexpr (LPR >= 8) x += dpp<0x141>(x);    // half rows mirrored
  if constexpr (LPR >= 16) x += dpp<0x140>(x);   // rows mirrored
  return x;
}

constexpr int ST_NT = 256;

// LPR lanes hold a channel's states, four each: a wave reads and writes whole runs of the state.
// A block takes `rows` rows of the batch, whose A it reads once.
template <typename T, int LPR>
__global__ __launch_bounds__(ST_NT) void scan_step_kernel(tops_gla_scan_step_args a, int rows,
                                                          int cb, int vec) {
  const int q = threadIdx.x % LPR, n0 = 4 * q;
  const int d = blockIdx.x % cb * (ST_NT / LPR) + threadIdx.x / LPR;
  const int b0 = blockIdx.x / cb * rows;
  const int D = (int)a.D, N = (int)a.N;
  const bool live = d < D;
  const int dd = live ? d : 0;
  const int grp = dd / (D / (int)a.G);
  const int nn = live ? min(4, N - n0) : 0;   // valid states of the lane
  const bool v4 = vec && nn == 4;
  float A[4] = {};
  if (v4) {
    const float4 w = *reinterpret_cast<const float4*>(a.A + (long)dd * N + n0);
    A[0] = w.x, A[1] = w.y, A[2] = w.z, A[3] = w.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] = i < nn ? a.A[(long)dd * N + n0 + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] *= 1.4426950408889634f;
  const float bias = a.delta_bias ? a.delta_bias[dd] : 0.f;
  const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
  const int b1 = min((int)a.batch, b0 + rows);
  for (int b = b0; b < b1; ++b) {
    const long slot = slot_of(a.slots_idx, a.idx64, b);
    const bool there = slot >= 0 && slot < a.slots;
    float y = 0.f, h[4] = {};
    float* s = a.state + (there ? slot : 0) * a.state_ss + (long)dd * N + n0;
    if (there) {
      if (v4) {
        const float4 w = *reinterpret_cast<const float4*>(s);
        h[0] = w.x, h[1] = w.y, h[2] = w.z, h[3] = w.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = i < nn ? s[i] : 0.f;
      }
    }
    const float u = to_f32(((const T*)a.u)[b * a.u_sb + dd]);
    float dt = to_f32(((const T*)a.delta)[b * a.delta_sb + dd]) + bias, sg;
    const float z = a.z ? to_f32(((const T*)a.z)[b * a.z_sb + dd]) : 0.f;
    const T* Bp = (const T*)a.B + b * a.B_sb + grp * a.B_sg + n0;
    const T* Cp = (const T*)a.C + b * a.C_sb + grp * a.C_sg + n0;
    float Bv[4], Cv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Bv[i] = i < nn ? to_f32(Bp[i]) : 0.f;
      Cv[i] = i < nn ? to_f32(Cp[i]) : 0.f;
    }
    if (a.softplus) softplus_sigmoid(dt, dt, sg);
    const float du = dt * u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = fmaf(__builtin_amdgcn_exp2f(A[i] * dt), h[i], du * Bv[i]);
      y = fmaf(Cv[i], h[i], y);
    }
    if (there) {
      if (v4) {
        *reinterpret_cast<float4*>(s) = make_float4(h[0], h[1], h[2], h[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < nn) s[i] = h[i];
      }
    }
    y = sum_adjacent<LPR>(nn > 0 ? y : 0.f);
    if (q == 0 && live) {
      y = fmaf(skip, u, y);
      if (a.z) y *= z * sigmoid(z);
      ((T*)a.y)[(long)b * D + d] = from_f32<T>(there ? y : 0.f);
    }
  }
}

template <typename T>
hipError_t scan_step(const tops_gla_scan_step_args& a, hipStream_t st) {
  const int N = (int)a.N;
  const int vec = N % 4 == 0 && a.state_ss % 4 == 0 && ((uintptr_t)a.state & 15) == 0 &&
                  ((uintptr_t)a.A & 15) == 0;
  const int lpr = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
  const int cb = (int)((a.D + ST_NT / lpr - 1) / (ST_NT / lpr));
  // rows of a block: A is read once for all of them, as long as the blocks fill the device
  int rows = 1;
  while (rows < 8 && (long)cb * ((a.batch + 2 * rows - 1) / (2 * rows)) >= 2048) rows *= 2;
  const dim3 grid((unsigned)(cb * ((a.batch + rows - 1) / rows)));
  switch (lpr) {
    case 1: hipLaunchKernelGGL((scan_step_kernel<T, 1>), grid, dim3(ST_NT), 0, st, a, rows, cb, vec); break;
    case 2: hipLaunchKernelGGL((scan_step_kernel<T, 2>), grid, dim3(ST_NT), 0, st, a, rows, cb, vec); break;
    case 4: hipLaunchKernelGGL((scan_step_kernel<T, 4>), grid, dim3(ST_NT), 0, st, a, rows, cb, vec); break;
    case 8: hipLaunchKernelGGL((scan_step_kernel<T, 8>), grid, dim3(ST_NT), 0, st, a, rows, cb, vec); break;
    default: hipLaunchKernelGGL((scan_step_kernel<T, 16>), grid, dim3(ST_NT), 0, st, a, rows, cb, vec);
  }
  return hipGetLastError();
}

// One thread per (row, VEC channels): the window moves up a row in place.
template <typename T, typename TW, int VEC>
__global__ __launch_bounds__(ST_NT) void conv_step_kernel(tops_gla_conv_step_args a, int cb) {
  const int D = (int)a.D, W = (int)a.W;
  const int c = (blockIdx.x % cb * ST_NT + threadIdx.x) * VEC, b = blockIdx.x / cb;
  if (c >= D) return;
  const long slot = slot_of(a.slots_idx, a.idx64, b);
  const bool there = slot >= 0 && slot < a.slots;
  float y[VEC] = {};
  if (there) {
    T* s = (T*)a.state + slot * a.state_ss + c;
    const TW* w = (const TW*)a.w + (long)c * W;
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = a.bias ? to_f32(((const TW*)a.bias)[c + e]) : 0.f;
    struct alignas(VEC * sizeof(T)) Raw { T v[VEC]; };
    Raw r[8];
    const Raw x = *reinterpret_cast<const Raw*>((const T*)a.x + b * a.x_sb + c);
#pragma unroll
    for (int j = 0; j < 8; ++j)   // the row that moves to j
      if (j < W) r[j] = j == W - 1 ? x : *reinterpret_cast<const Raw*>(s + (long)(j + 1) * D);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < W) {
        *reinterpret_cast<Raw*>(s + (long)j * D) = r[j];
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = fmaf(to_f32(w[e * W + j]), to_f32(r[j].v[e]), y[e]);
      }
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (a.silu) y[e] *= sigmoid(y[e]);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) ((T*)a.y)[(long)b * D + c + e] = from_f32<T>(y[e]);
}

template <typename T, typename TW>
hipError_t conv_step(const tops_gla_conv_step_args& a, hipStream_t st) {
  // four channels a thread where the rows allow it (a step has few threads to begin with)
  const bool vec = a.D % 4 == 0 && a.x_sb % 4 == 0 && a.state_ss % 4 == 0 &&
                   ((uintptr_t)a.x & (4 * sizeof(T) - 1)) == 0 &&
                   ((uintptr_t)a.state & (4 * sizeof(T) - 1)) == 0;
  const long per = vec ? 4 : 1;
  const int cb = (int)((a.D + ST_NT * per - 1) / (ST_NT * per));
  const dim3 grid((unsigned)(cb * a.batch));
  if (vec)
    hipLaunchKernelGGL((conv_step_kernel<T, TW, 4>), grid, dim3(ST_NT), 0, st, a, cb);
  else
    hipLaunchKernelGGL((conv_step_kernel<T, TW, 1>), grid, dim3(ST_NT), 0, st, a, cb);
  return hipGetLastError();
}

}  // namespace

hipError_t run_scan_step(const tops_gla_scan_step_args& a, hipStream_t st) {
  if (a.batch == 0 || a.D == 0) return hipSuccess;
  return a.dtype == DT_BF16 ? scan_step<bf16>(a, st) : scan_step<float>(a, st);
}

hipError_t run_conv_step(const tops_gla_conv_step_args& a, hipStream_t st) {
  if (a.batch == 0 || a.D == 0) return hipSuccess;
  if (a.dtype == DT_BF16)
    return a.w_dtype == DT_BF16 ? conv_step<bf16, bf16>(a, st) : conv_step<bf16, float>(a, st);
  return a.w_dtype == DT_BF16 ? conv_step<float, bf16>(a, st) : conv_step<float, float>(a, st);
}

}  // namespace tops
