// The single-token forms: one step of the selective scan and of its convolution for each row of
// a serving batch, the states updated in place (include/tops_gla_ssm.h).
//
// Both are bound by the states' traffic (a row's state is read and written once), and for a few
// rows by the launch. MI355X: scan, 128 rows of 4096 channels, N 16: 15.8 us (4.5 TB/s), one row of
// 2048 channels 3.2; convolution, W 4: 4.1 and 2.4.
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
// A block takes up to U rows of the batch, whose A it reads once and whose loads are all sent
// before the first row is computed.
template <typename T, int LPR, int U>
__global__ __launch_bounds__(ST_NT) void scan_step_kernel(tops_gla_scan_step_args a, int cb,
                                                          int vec, int vecbc) {
  const int q = threadIdx.x % LPR, n0 = 4 * q;
  const int d = blockIdx.x % cb * (ST_NT / LPR) + threadIdx.x / LPR;
  const int b0 = blockIdx.x / cb * U;
  const int D = (int)a.D, N = (int)a.N;
  const bool live = d < D;
  // a branch of the whole launch: selects for every N cost the 128 rows below 1.8 us
  const bool pad = N % 4 != 0;
  const int dd = live ? d : 0;
  const int grp = a.G == 1 ? 0 : dd / (D / (int)a.G);
  const int nn = live ? min(4, N - n0) : 0;   // valid states of the lane
  const bool v4 = vec && nn == 4, v4bc = vecbc && nn == 4;
  const int rows = min(U, (int)a.batch - b0);
  float h[U][4], u[U], dt[U], z[U], B[U][4], C[U][4];
  float* s[U];
  bool there[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int b = b0 + min(k, rows - 1);
    const long slot = slot_of(a.slots_idx, a.idx64, b);
    there[k] = k < rows && slot >= 0 && slot < a.slots;
    s[k] = a.state + (there[k] ? slot : 0) * a.state_ss + (long)dd * N + n0;
    u[k] = to_f32(((const T*)a.u)[b * a.u_sb + dd]);
    dt[k] = to_f32(((const T*)a.delta)[b * a.delta_sb + dd]);
    z[k] = a.z ? to_f32(((const T*)a.z)[b * a.z_sb + dd]) : 0.f;
    const T* Bp = (const T*)a.B + b * a.B_sb + grp * a.B_sg + n0;
    const T* Cp = (const T*)a.C + b * a.C_sb + grp * a.C_sg + n0;
    if (v4bc) {
      load_four(Bp, B[k]);
      load_four(Cp, C[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        B[k][i] = i < nn ? to_f32(Bp[i]) : 0.f;
        C[k][i] = i < nn ? to_f32(Cp[i]) : 0.f;
      }
    }
    if (a.slots > 0 && v4) {   // slot 0 in the place of one that is not there
      load_four((const float*)s[k], h[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) h[k][i] = a.slots > 0 && i < nn ? s[k][i] : 0.f;
    }
  }
  float A[4];
  if (v4) {
    load_four(a.A + (long)dd * N + n0, A);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] = i < nn ? a.A[(long)dd * N + n0 + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) A[i] = scaled_a(A[i]);
  const float bias = a.delta_bias ? a.delta_bias[dd] : 0.f;
  const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float t = dt[k] + bias, y = 0.f;
    if (a.softplus) t = softplus(t);
    const float du = t * u[k];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[k][i] = fmaf(__builtin_amdgcn_exp2f(A[i] * t), h[k][i], du * B[k][i]);
      if (!pad) y = fmaf(C[k][i], h[k][i], y);
    }
    if (pad)   // an infinite u makes a NaN of what fills a lane's four states
#pragma unroll
      for (int i = 0; i < 4; ++i) y = i < nn ? fmaf(C[k][i], h[k][i], y) : y;
    if (there[k]) {
      if (v4) {
        st16_nt(s[k], 0, __builtin_bit_cast(uint4, make_float4(h[k][0], h[k][1], h[k][2], h[k][3])));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < nn) s[k][i] = h[k][i];
      }
    }
    y = sum_adjacent<LPR>(nn > 0 ? y : 0.f);
    if (q == 0 && live && k < rows) {
      y = fmaf(skip, u[k], y);
      if (a.z) y *= z[k] * sigmoid(z[k]);
      ((T*)a.y)[(long)(b0 + k) * D + d] = from_f32<T>(there[k] ? y : 0.f);
    }
  }
}

template <typename T, int LPR>
hipError_t scan_step_lanes(const tops_gla_scan_step_args& a, int vec, int vecbc, hipStream_t st) {
  const int cb = (int)((a.D + ST_NT / LPR - 1) / (ST_NT / LPR));
  // two rows a block as long as the blocks fill the device (128 rows of 4096 channels, N 16: 18.0
  // us with one, 17.0 with two, 20.0 with four; 15.8 with stores past the L2)
  if (cb * ((a.batch + 1) / 2) >= 1024)
    hipLaunchKernelGGL((scan_step_kernel<T, LPR, 2>), dim3((unsigned)(cb * ((a.batch + 1) / 2))),
                       dim3(ST_NT), 0, st, a, cb, vec, vecbc);
  else
    hipLaunchKernelGGL((scan_step_kernel<T, LPR, 1>), dim3((unsigned)(cb * a.batch)), dim3(ST_NT), 0,
                       st, a, cb, vec, vecbc);
  return hipGetLastError();
}

template <typename T>
hipError_t scan_step(const tops_gla_scan_step_args& a, hipStream_t st) {
  const int N = (int)a.N, es = (int)sizeof(T);
  const int vec = N % 4 == 0 && a.state_ss % 4 == 0 && ((uintptr_t)a.state & 15) == 0 &&
                  ((uintptr_t)a.A & 15) == 0;
  const int vecbc = a.B_sb % 4 == 0 && a.C_sb % 4 == 0 && a.B_sg % 4 == 0 && a.C_sg % 4 == 0 &&
                    ((uintptr_t)a.B & (4 * es - 1)) == 0 && ((uintptr_t)a.C & (4 * es - 1)) == 0;
  if (N <= 4) return scan_step_lanes<T, 1>(a, vec, vecbc, st);
  if (N <= 8) return scan_step_lanes<T, 2>(a, vec, vecbc, st);
  if (N <= 16) return scan_step_lanes<T, 4>(a, vec, vecbc, st);
  if (N <= 32) return scan_step_lanes<T, 8>(a, vec, vecbc, st);
  return scan_step_lanes<T, 16>(a, vec, vecbc, st);
}

// One thread per (row, VEC channels): the window moves up a row in place.
template <typename T, typename TW, int VEC, int W>
__global__ __launch_bounds__(ST_NT) void conv_step_kernel(tops_gla_conv_step_args a, int cb) {
  const int D = (int)a.D;
  const int c = (blockIdx.x % cb * ST_NT + threadIdx.x) * VEC, b = blockIdx.x / cb;
  if (c >= D) return;
  struct alignas(VEC * sizeof(T)) Raw { T v[VEC]; };
  const Raw x = *reinterpret_cast<const Raw*>((const T*)a.x + b * a.x_sb + c);
  float w[VEC * W], y[VEC] = {};
  const TW* wp = (const TW*)a.w + (long)c * W;
  if constexpr (VEC == 4) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float four[4];
      load_four(wp + 4 * j, four);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * j + e] = four[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC * W; ++j) w[j] = to_f32(wp[j]);
  }
  if (a.bias)
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = to_f32(((const TW*)a.bias)[c + e]);
  const long slot = slot_of(a.slots_idx, a.idx64, b);
  if (slot >= 0 && slot < a.slots) {
    T* s = (T*)a.state + slot * a.state_ss + c;
    Raw r[W];   // the rows that move to 0 .. W - 1
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) r[j] = *reinterpret_cast<const Raw*>(s + (long)(j + 1) * D);
    r[W - 1] = x;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      *reinterpret_cast<Raw*>(s + (long)j * D) = r[j];
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = fmaf(w[e * W + j], to_f32(r[j].v[e]), y[e]);
    }
    if (a.silu)
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] *= sigmoid(y[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = 0.f;
  }
  Raw o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.v[e] = from_f32<T>(y[e]);
  *reinterpret_cast<Raw*>((T*)a.y + (long)b * D + c) = o;
}

template <typename T, typename TW, int W>
hipError_t conv_step_width(const tops_gla_conv_step_args& a, hipStream_t st) {
  // four channels a thread where the rows allow it (a step has few threads to begin with)
  const auto at = [](const void* p, size_t by) { return ((uintptr_t)p & (by - 1)) == 0; };
  const bool vec = a.D % 4 == 0 && a.x_sb % 4 == 0 && a.state_ss % 4 == 0 &&
                   at(a.x, 4 * sizeof(T)) && at(a.state, 4 * sizeof(T)) && at(a.y, 4 * sizeof(T)) &&
                   at(a.w, 4 * sizeof(TW));
  const long per = vec ? 4 : 1;
  const int cb = (int)((a.D + ST_NT * per - 1) / (ST_NT * per));
  const dim3 grid((unsigned)(cb * a.batch));
  if (vec)
    hipLaunchKernelGGL((conv_step_kernel<T, TW, 4, W>), grid, dim3(ST_NT), 0, st, a, cb);
  else
    hipLaunchKernelGGL((conv_step_kernel<T, TW, 1, W>), grid, dim3(ST_NT), 0, st, a, cb);
  return hipGetLastError();
}

template <typename T, typename TW>
hipError_t conv_step(const tops_gla_conv_step_args& a, hipStream_t st) {
  switch (a.W) {
    case 1: return conv_step_width<T, TW, 1>(a, st);
    case 2: return conv_step_width<T, TW, 2>(a, st);
    case 3: return conv_step_width<T, TW, 3>(a, st);
    case 4: return conv_step_width<T, TW, 4>(a, st);
    case 5: return conv_step_width<T, TW, 5>(a, st);
    case 6: return conv_step_width<T, TW, 6>(a, st);
    case 7: return conv_step_width<T, TW, 7>(a, st);
    default: return conv_step_width<T, TW, 8>(a, st);
  }
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
