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
  int ntiles, tiles_g;   // channel tiles of 64 in all and of a group
  int btiles;            // channel tiles of the backward's blocks
  int pieces;            // pieces of a sequence (fixed length)
  int multi;             // some sequence has more than one piece
  long npieces, tokens;
  const float* at;       // A log2(e), [NP][D], behind the rows of bc
  float *part_bc, *part_a, *part_d;   // the backward's shares
};
int scan_state_pad(int N);       // N rounded up to 8, 16, 32 or 64
int scan_bwd_channels(int N);    // channels of a block of the backward
int scan_bwd_threads(int N);     // and threads
int scan_chunk();                // tokens between the states kept for the backward
hipError_t run_selective_scan(const ScanParams& p, bool backward, hipStream_t st);

hipError_t run_scan_step(const tops_gla_scan_step_args& a, hipStream_t st);
hipError_t run_conv_step(const tops_gla_conv_step_args& a, hipStream_t st);

hipError_t run_causal_conv_fwd(const tops_gla_conv_args& a, hipStream_t st);
hipError_t run_causal_conv_bwd(const tops_gla_conv_args& a, hipStream_t st);
long causal_conv_part_rows(long tokens, long D);   // rows of (W + 1) D partial weight gradients

hipError_t run_qk_norm_rope(const tops_gla_qk_args& a, bool backward, hipStream_t st);
long qk_norm_rope_part_rows(long tokens);  // rows of 2 D partial weight gradients
long qk_norm_rope_blocks(long tokens, long heads);   // of the forward, 256 threads each

// Four elements at an address that is a multiple of theirs.
__device__ __forceinline__ void load_four(const float* p, float (&x)[4]) {
  const float4 w = *reinterpret_cast<const float4*>(p);
  x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
}
__device__ __forceinline__ void load_four(const bf16* p, float (&x)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
}

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

// A log2(e). -inf (a state that is forgotten at once) stays finite: where delta' is 0 the state is
// kept, as for every other A, and a token past a sequence's end has a delta' of 0.
__device__ __forceinline__ float scaled_a(float a) {
  a *= 1.4426950408889634f;
  return a < -3.4028235e38f ? -3.4028235e38f : a;
}

// 1 / (1 + e^-x), with the hardware exponential and reciprocal (1 ulp each); 0 and 1 at the ends.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// log(1 + e^x), and its derivative. With w = e^-|x| and u = 1 + w rounded, log(1 + w) = log(u) +
// (w - (u - 1)) / u to second order, which keeps the relative accuracy of a small result; the
// exponent's rounding is put back to first order, as it grows with |x|. w is cut at |x| = 104,
// where float32 has nothing left of it, so that infinities need no case of their own (the minimum
// passes a NaN on).
__device__ __forceinline__ float exp_minus_abs(float x) {
  const float L2E = 1.4426950408889634f, L2E_LO = 1.9259629911266175e-8f;
  const float ax = __builtin_elementwise_minimum(fabsf(x), 104.f);
  const float e = -ax * L2E;
  const float r = fmaf(-ax, L2E_LO, fmaf(-ax, L2E, -e));   // what the product lost
  const float w = __builtin_amdgcn_exp2f(e);
  return fmaf(w * r, 0.6931471805599453f, w);
}
__device__ __forceinline__ void softplus_sigmoid(float x, float& sp, float& sg) {
  const float w = exp_minus_abs(x), u = 1.f + w, iu = __builtin_amdgcn_rcpf(u);
  sp = fmaxf(x, 0.f) +
       fmaf(w - (u - 1.f), iu, __builtin_amdgcn_logf(u) * 0.6931471805599453f);
  sg = x >= 0.f ? iu : w * iu;
}
// log(1 + e^x) alone: the second-order term is at most half a step of u, so that 1 - w / 2 does
// for its 1 / u.
__device__ __forceinline__ float softplus(float x) {
  const float w = exp_minus_abs(x), u = 1.f + w;
  return fmaxf(x, 0.f) + fmaf(w - (u - 1.f), fmaf(-0.5f, w, 1.f),
                              __builtin_amdgcn_logf(u) * 0.6931471805599453f);
}

}  // namespace tops
