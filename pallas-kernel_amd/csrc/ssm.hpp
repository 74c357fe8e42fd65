// Launch interface and device helpers of the selective state space operators.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/tops_gla.h"
#include "../../include/tops_gla_ssm.h"
#include "common.hpp"
#include "kernels.hpp"

namespace tops {

// Records the calling thread's error message (capi.hip); returns `code`.
int set_error(int code, const char* msg);

struct ScanParams {
  tops_gla_scan_args a;
  int ntiles, tiles_g;   // channel tiles in all and of a group
  int pieces;            // pieces of a sequence (fixed length)
  int multi;             // some sequence has more than one piece
  int vec;               // rows allow wide loads and stores
  long npieces, tokens;
  float *part_bc, *part_a, *part_d;   // the backward's shares
};
int scan_state_pad(int N);       // N rounded up to 16, 32 or 64
int scan_tile_channels(int N);   // channels of a block
hipError_t run_selective_scan(const ScanParams& p, bool backward, hipStream_t st);

hipError_t run_scan_step(const tops_gla_scan_step_args& a, hipStream_t st);
hipError_t run_conv_step(const tops_gla_conv_step_args& a, hipStream_t st);

hipError_t run_causal_conv_fwd(const tops_gla_conv_args& a, hipStream_t st);
hipError_t run_causal_conv_bwd(const tops_gla_conv_args& a, hipStream_t st);
long causal_conv_part_rows(long tokens);   // rows of (W + 1) D partial weight gradients

hipError_t run_qk_norm_rope(const tops_gla_qk_args& a, bool backward, hipStream_t st);
long qk_norm_rope_part_rows(long tokens);  // rows of 2 D partial weight gradients

// Value of a lane of the same row of 16 (CTRL: 0x120 + r rotates right by r).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(
      (uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// a + a of the other half wave in lanes 0-31, the same of b in lanes 32-63.
__device__ __forceinline__ float swap32_add(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// a summed over each pair of rows of 16 lanes in the even rows, b in the odd ones.
__device__ __forceinline__ float swap16_add(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// v summed over the CPW lanes of consecutive channels (lane bits below log2 CPW): v[0..3] go to
// out[n0 .. n0 + 3], v[4..7] to out[np + n0 ..].
template <int CPW>
__device__ __forceinline__ void sum_channels(float (&v)[8], int lane, float* out, int n0, int np) {
  if constexpr (CPW == 16) {
    const bool b3 = lane & 8, b2 = lane & 4;
    float r[4], s[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // lanes with bit 3 set take dC, the others dB
      const float x = v[i] + dpp<0x128>(v[i]), y = v[4 + i] + dpp<0x128>(v[4 + i]);
      r[i] = b3 ? y : x;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // bit 2: the upper two states (half rows mirrored)
      const float x = r[i] + dpp<0x141>(r[i]), y = r[2 + i] + dpp<0x141>(r[2 + i]);
      s[i] = b2 ? y : x;
      s[i] += dpp<0xb1>(s[i]);      // quad_perm [1, 0, 3, 2]
      s[i] += dpp<0x4e>(s[i]);      // quad_perm [2, 3, 0, 1]
    }
    if ((lane & 3) == 0)
      *reinterpret_cast<float2*>(out + (b3 ? np : 0) + n0 + (b2 ? 2 : 0)) = make_float2(s[0], s[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (CPW >= 8) v[i] += dpp<0x141>(v[i]);
      v[i] += dpp<0xb1>(v[i]);
      v[i] += dpp<0x4e>(v[i]);
    }
    if ((lane & (CPW - 1)) == 0) {
      *reinterpret_cast<float4*>(out + n0) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(out + np + n0) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
}

// 1 / (1 + e^-x), with the hardware exponential and reciprocal (1 ulp each); 0 and 1 at the ends.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// log(1 + e^x) and its derivative. With w = e^-|x| and u = 1 + w rounded, log(1 + w) = log(u) +
// (w - (u - 1)) / u to second order, which keeps the relative accuracy of a small result; the
// exponent's rounding is put back to first order, as it grows with |x|.
__device__ __forceinline__ void softplus_sigmoid(float x, float& sp, float& sg) {
  const float L2E = 1.4426950408889634f, L2E_LO = 1.9259629911266175e-8f;
  const float ax = fabsf(x);
  const float e = -ax * L2E;
  float r = -fmaf(ax, L2E, e);            // what the product lost
  r = fmaf(-ax, L2E_LO, r);
  float w = __builtin_amdgcn_exp2f(e);
  w = w > 0.f ? fmaf(w, r * 0.6931471805599453f, w) : 0.f;   // |x| = inf: r is NaN, w is 0
  const float u = 1.f + w, iu = __builtin_amdgcn_rcpf(u);
  const float l = fmaf(w - (u - 1.f), iu, __builtin_amdgcn_logf(u) * 0.6931471805599453f);
  sp = x != x ? x : fmaxf(x, 0.f) + l;
  sg = x != x ? x : x >= 0.f ? iu : w * iu;
}

}  // namespace tops
