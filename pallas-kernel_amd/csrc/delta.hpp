// Launch interface and device helpers of the gated delta rule and of the layer norm.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/tops_gla.h"
#include "../../include/tops_gla_delta.h"
#include "common.hpp"
#include "kernels.hpp"
#include "ssm.hpp"

namespace tops {

hipError_t run_layer_norm_fwd(const tops_gla_layer_norm_args& a, hipStream_t st);
hipError_t run_layer_norm_bwd(const tops_gla_layer_norm_args& a, hipStream_t st);
long layer_norm_part_rows(long rows, long D, int dtype);   // rows of 2 D partial sums

hipError_t run_delta_step(const tops_gla_delta_step_args& a, hipStream_t st);

// N consecutive elements at any address of theirs: the wide loads and stores need no alignment
// beyond the element's.
template <typename T, int N>
struct Run {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Run<T, N> get_run(const T* p) {
  return *reinterpret_cast<const Run<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void put_run(T* p, const float (&x)[N], int n = N) {
  if (n >= N) {
    Run<T, N> r;
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = from_f32<T>(x[e]);
    *reinterpret_cast<Run<T, N>*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) p[e] = from_f32<T>(x[e]);
  }
}

// The 8 elements from column c on, zeros from `cols` on, of the 8 that were loaded from
// min(c, cols - 8).
__device__ __forceinline__ Run<bf16, 8> cut_run(const Run<bf16, 8>& r, int c, int cols) {
  uint4 x = __builtin_bit_cast(uint4, r);
  if (cols % 8) {   // the same for all lanes
    const int s = max(0, min(c - (cols - 8), 8));
    if (s & 4) x = make_uint4(x.z, x.w, 0, 0);
    if (s & 2) x = make_uint4(x.y, x.z, x.w, 0);
    if (s & 1)
      x = make_uint4(x.x >> 16 | x.y << 16, x.y >> 16 | x.z << 16, x.z >> 16 | x.w << 16,
                     x.w >> 16);
  }
  return __builtin_bit_cast(Run<bf16, 8>, mask16(x, c < cols ? ~0u : 0u));
}
__device__ __forceinline__ Run<float, 8> cut_run(const Run<float, 8>& r, int c, int cols) {
  Run<float, 8> x = r;
  if (cols % 8) {
    const int s = max(0, min(c - (cols - 8), 8));
#pragma unroll
    for (int b = 4; b > 0; b >>= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] = s & b ? (e + b < 8 ? x.v[e + b] : 0.f) : x.v[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x.v[e] = c < cols ? x.v[e] : 0.f;
  return x;
}

// Element i of a tensor of either type.
__device__ __forceinline__ float get_any(const void* p, int dtype, long i) {
  return dtype == DT_BF16 ? to_f32(((const bf16*)p)[i]) : ((const float*)p)[i];
}
__device__ __forceinline__ void put_any(void* p, int dtype, long i, float x) {
  if (dtype == DT_BF16)
    ((bf16*)p)[i] = from_f32<bf16>(x);
  else
    ((float*)p)[i] = x;
}

constexpr float DELTA_L2_EPS = 1e-6f;

// e^g as the log decay that the kernels work with: -inf (a state that is forgotten) stays finite,
// so that differences of its sums do; e^-10000 is 0 all the same.
__device__ __forceinline__ float log_decay(float g) { return g < -1e4f ? -1e4f : g; }

// ---------------------------------------------------------------------------
// The chunked form
// ---------------------------------------------------------------------------

// Tokens of a chunk: 64 in bfloat16, and 32 in float32, whose tiles take twice the LDS.
template <typename T>
constexpr int delta_c() {
  return sizeof(T) == 2 ? 64 : 32;
}
inline int delta_chunk_of(int dtype) { return dtype == DT_BF16 ? 64 : 32; }
template <typename T>
constexpr int delta_blocks() {   // lower 32 x 32 blocks of a tile of C x C
  return delta_c<T>() == 64 ? 3 : 1;
}
__device__ __forceinline__ constexpr int tri_block(int u, int w) { return u * (u + 1) / 2 + w; }
constexpr int delta_key_pad(long K) { return K <= 64 ? 64 : K <= 128 ? 128 : 256; }
// Threads of a block: two waves for 16 tokens of a chunk, a wave for 32 padded keys.
constexpr int delta_grad_threads(int dtype) { return dtype == DT_BF16 ? 512 : 256; }
constexpr int delta_fold_threads(int KP) { return 2 * KP; }

// Per chunk and value head ("unit"): vectors over the chunk's tokens, [7][C] float and [C] double,
//   e^G / |k|, e^{G_C - G} / |k|, beta, 1 / |k|, e^G, e^{G_C - G}, 1 / |q|
// (norms 1 without l2norm) and G, the sums of the log decays (in 64 bits: differences of it go into
// exponentials), and the first token whose k, g or beta is not finite (C: none), from which on the
// chunk counts as empty but for a NaN in e^G and e^{G_C - G}, which makes its outputs, the state after
// the chunk, and gradients NaN; then, in the operands' type, three parts of it where that is bfloat16,
//   Tm the inverse of 1 + tril(beta k k^T decay), P the masked and scaled scores, both as the lower
// of their 32 x 32 blocks (0, 0), (1, 0), (1, 1);
// and, for the backward, in two such parts side by side in a row, N [V][2][C] the written values and
// S [V][2][KP] the state before the chunk.
struct DeltaParams {
  tops_gla_delta_args a;   // 8 <= K, 8 <= V
  int C, KP;   // tokens of a chunk, padded keys
  char *vec, *Tm, *P, *N, *S;   // in keep, the last three with `train`
  char *dS, *Y;                 // in ws, as S and N: the gradient of the state after the chunk, of the
                                // system's right side
  // where a sequence has several segments, for each of all segments and value heads: the state
  // after it [K][V] (E) or the gradient of the state before it (dE), float32, and what it makes of
  // a state before it, [KP][KP] (M, and Mt its transpose), in the order of the fold's operands, parts as Tm's
  float *E, *dE;
  char *M, *Mt;
  int multi;
  long vec_bytes, tri_bytes, map_bytes, keep_bytes, ws_bytes;
};
// The layout for given sizes; pointers from base addresses that may be NULL.
DeltaParams delta_layout(const tops_gla_delta_sizes& z, void* keep, void* ws);
hipError_t run_delta_prep(const DeltaParams& p, hipStream_t st);
hipError_t run_delta_scan(const DeltaParams& p, bool backward, hipStream_t st);
hipError_t run_delta_grad(const DeltaParams& p, hipStream_t st);

struct ChunkAt {
  int b, t, len;   // batch row, first token in it, tokens
};
__device__ __forceinline__ ChunkAt delta_chunk_at(const tops_gla_delta_args& a, int C, int c) {
  ChunkAt x;
  if (a.seqs) {
    const int* cc = a.seqs + a.nseq + 1;
    int lo = 0, hi = (int)a.nseq - 1;   // the last sequence whose first chunk is not behind c
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (cc[m] <= c) lo = m; else hi = m - 1;
    }
    x.b = 0;
    x.t = a.seqs[lo] + (c - cc[lo]) * C;
    x.len = min(C, a.seqs[lo + 1] - x.t);
  } else {
    const int nt = (int)((a.T + C - 1) / C);
    x.b = c / nt;
    x.t = (c - x.b * nt) * C;
    x.len = min(C, (int)a.T - x.t);
  }
  return x;
}

__device__ __forceinline__ float* delta_vec(const DeltaParams& p, long unit) {
  return (float*)(p.vec + unit * p.vec_bytes);
}
__device__ __forceinline__ int* delta_first(const DeltaParams& p, long unit) {
  return (int*)(p.vec + unit * p.vec_bytes + 36 * p.C);
}
__device__ __forceinline__ double* delta_gsum(const DeltaParams& p, long unit) {
  return (double*)(p.vec + unit * p.vec_bytes + 28 * p.C);
}

template <typename T>
__device__ __forceinline__ Frag<T> frag_of(const Run<T, 8>& r) {
  return __builtin_bit_cast(Frag<T>, r);
}
template <typename T>
__device__ __forceinline__ Frag<T> frag_of(const float (&x)[8]);
template <>
__device__ __forceinline__ Frag<float> frag_of<float>(const float (&x)[8]) {
  Frag<float> f;
  f.a = make_float4(x[0], x[1], x[2], x[3]);
  f.b = make_float4(x[4], x[5], x[6], x[7]);
  return f;
}
template <>
__device__ __forceinline__ Frag<bf16> frag_of<bf16>(const float (&x)[8]) {
  Frag<bf16> f;
  f.d = make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]),
                   pack2_bf16(x[6], x[7]));
  return f;
}
__device__ __forceinline__ void values_of(const Frag<float>& f, float (&x)[8]) {
  x[0] = f.a.x, x[1] = f.a.y, x[2] = f.a.z, x[3] = f.a.w;
  x[4] = f.b.x, x[5] = f.b.y, x[6] = f.b.z, x[7] = f.b.w;
}
__device__ __forceinline__ void values_of(const Frag<bf16>& f, float (&x)[8]) {
  const uint32_t w[4] = {f.d.x, f.d.y, f.d.z, f.d.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
}
template <typename T>
__device__ __forceinline__ void st_frag(T* p, const Frag<T>& f) {   // 16-byte aligned
  __builtin_memcpy(__builtin_assume_aligned(p, 16), &f, sizeof(f));
}

// A float operand in N parts of its products' type, the largest first. In bfloat16 three parts hold
// all 24 bits of a float: states and what they are made of go through such products, so that a state
// is as exact in bfloat16 calls as float32 sums allow. Two parts are 2^-17 of the value off at most
// (half a step of a remainder that is half a step itself): what goes into a result of bfloat16.
template <typename T, int N>
struct Split {
  Frag<T> p[N];
};
template <typename T>
constexpr int WHOLE = sizeof(T) == 2 ? 3 : 1;
template <typename T>
constexpr int TWO = sizeof(T) == 2 ? 2 : 1;
template <typename T>
using Whole = Split<T, WHOLE<T>>;
template <typename T>
using Two = Split<T, TWO<T>>;

template <typename T, int N>
__device__ __forceinline__ Split<T, N> split_of(const float (&x)[8]) {
  Split<T, N> s;
  s.p[0] = frag_of<T>(x);
  if constexpr (N > 1) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int i = 1; i < N; ++i) {
      uint4& d = s.p[i - 1].d;
      // hides the packed words, whose halves the compiler would otherwise convert once more
      asm("" : "+v"(d.x), "+v"(d.y), "+v"(d.z), "+v"(d.w));
      float h[8];
      values_of(s.p[i - 1], h);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] -= h[e];
      s.p[i] = frag_of<T>(r);
    }
  }
  return s;
}
template <typename T, int N>
__device__ __forceinline__ void sum_of(const Split<T, N>& s, float (&x)[8]) {
  values_of(s.p[N - 1], x);
#pragma unroll
  for (int i = N - 2; i >= 0; --i) {
    float h[8];
    values_of(s.p[i], h);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += h[e];
  }
}
template <typename T>
__device__ __forceinline__ Two<T> two_of(const Whole<T>& w) {
  Two<T> s;
#pragma unroll
  for (int i = 0; i < TWO<T>; ++i) s.p[i] = w.p[i];
  return s;
}
// The products of the parts, the smallest first; those of two small parts that are below what the
// others leave off are left out.
template <typename T, int N>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<T>& a, const Split<T, N>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i) mma(acc, a, b.p[i]);
}
template <typename T, int N>
__device__ __forceinline__ void mma(f32x4& acc, const Split<T, N>& a, const Frag<T>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i) mma(acc, a.p[i], b);
}
template <typename T, int N>
__device__ __forceinline__ void mma(f32x4& acc, const Split<T, N>& a, const Split<T, N>& b) {
#pragma unroll
  for (int s = N - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i) mma(acc, a.p[i], b.p[s - i]);
}

// Output tiles come in pairs (h = 0, 1) of 32 rows: row 4 g + r of tile h stands for row
// 8 g + 4 h + r, so that a lane's accumulators of both tiles are 8 consecutive rows of its column,
// which is what an operand fragment over those rows holds: a result becomes the next product's
// operand without leaving its lane. The row that lane i supplies to tile h as the first operand:
__device__ __forceinline__ int pair_row(int lane, int h) {
  return 8 * ((lane & 15) >> 2) + 4 * h + (lane & 3);
}
// The same rows read from a row-major [k][row] tile in LDS (M at element [k0][row0]).
__device__ __forceinline__ Frag<bf16> ld_pair_t(const bf16* M, int P, int lane, int h) {
  const int g = lane >> 4, j = lane & 15;
  const bf16* p1 = M + (8 * g + (j >> 2)) * P + 8 * (j & 3) + 4 * h;
  const s4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s4_t*)(p1));
  const s4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s4_t*)(p1 + 4 * P));
  const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
  Frag<bf16> f;
  f.d = make_uint4(ua.x, ua.y, ub.x, ub.y);
  return f;
}
__device__ __forceinline__ Frag<float> ld_pair_t(const float* M, int P, int lane, int h) {
  const float* p = M + (8 * (lane >> 4)) * P + pair_row(lane, h);
  Frag<float> f;
  f.a = make_float4(p[0], p[P], p[2 * P], p[3 * P]);
  f.b = make_float4(p[4 * P], p[5 * P], p[6 * P], p[7 * P]);
  return f;
}
// Split fragments of a tile whose parts lie `step` elements apart.
template <typename T, int N>
__device__ __forceinline__ Split<T, N> ld_split(const T* tile, int step, int off) {
  Split<T, N> s;
#pragma unroll
  for (int i = 0; i < N; ++i) s.p[i] = ld_frag(tile + i * step + off);
  return s;
}
template <typename T, int N>
__device__ __forceinline__ Split<T, N> ld_split_t(const T* tile, int step, int P, int lane, int h) {
  Split<T, N> s;
#pragma unroll
  for (int i = 0; i < N; ++i) s.p[i] = ld_pair_t(tile + i * step, P, lane, h);
  return s;
}
// The 8 values of a lane in a pair of accumulators.
__device__ __forceinline__ void pair_values(const f32x4& a, const f32x4& b, float (&x)[8]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = a[r], x[4 + r] = b[r];
}

// A value that is there whatever becomes of it: a choice made with it needs no branch around what it
// comes from (the compiler puts LDS reads and exponentials into such branches, one wait for each).
__device__ __forceinline__ float pinned(float x) {
  asm volatile("" : "+v"(x));
  return x;
}
// 8 floats in a row in LDS, 16-byte aligned.
__device__ __forceinline__ void ld_eight(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = pinned(a.x), x[1] = pinned(a.y), x[2] = pinned(a.z), x[3] = pinned(a.w);
  x[4] = pinned(b.x), x[5] = pinned(b.y), x[6] = pinned(b.z), x[7] = pinned(b.w);
}
// e^{sign (G - Gj)} for 8 tokens j in a row.
template <typename T>
__device__ __forceinline__ void decays(double G, const double* Gj, float sign, float (&d)[8]) {
  double y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = G - Gj[e];
#pragma unroll
  for (int e = 0; e < 8; ++e) d[e] = pinned(gexp<T>(sign * (float)y[e]));
}

// 8 elements at any address of theirs, as whole registers (loads of them are not taken apart).
template <typename T>
struct Piece;
template <>
struct Piece<bf16> {
  typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
  u32x4_t x;
  __device__ __forceinline__ void get(const void* base, uint32_t off) {
    x = *reinterpret_cast<const Any*>((const char*)base + off);
  }
  // A sum that goes into the sign where an exponent has all its bits.
  static constexpr uint32_t SIGNS = 0x80008000u;
  __device__ __forceinline__ uint32_t full() const {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (x[i] & ~SIGNS) + 0x00800080u;
    return r;
  }
  __device__ __forceinline__ Frag<bf16> frag() const {
    Frag<bf16> f;
    f.d = make_uint4(x[0], x[1], x[2], x[3]);
    return f;
  }
};
template <>
struct Piece<float> {
  typedef float Any __attribute__((ext_vector_type(4), aligned(4)));
  f32x4 x, y;
  __device__ __forceinline__ void get(const void* base, uint32_t off) {
    x = *reinterpret_cast<const Any*>((const char*)base + off);
    y = *reinterpret_cast<const Any*>((const char*)base + off + 16);
  }
  static constexpr uint32_t SIGNS = 0x80000000u;
  __device__ __forceinline__ uint32_t full() const {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r |= ((__float_as_uint(x[i]) & ~SIGNS) + 0x00800000u) |
           ((__float_as_uint(y[i]) & ~SIGNS) + 0x00800000u);
    return r;
  }
  __device__ __forceinline__ Frag<float> frag() const {
    Frag<float> f;
    f.a = make_float4(x[0], x[1], x[2], x[3]);
    f.b = make_float4(y[0], y[1], y[2], y[3]);
    return f;
  }
};
template <typename T>
using Eight = Run<T, 8>;
template <typename T>
__device__ __forceinline__ Frag<T> cut_frag(const Frag<T>& f, int c, int cols) {
  return __builtin_bit_cast(Frag<T>, cut_run(__builtin_bit_cast(Eight<T>, f), c, cols));
}

// A [C][W] tile on its way to LDS in pieces of 8 elements. The loads have no conditions, so that
// they are all on their way at once: a piece past the tile's rows or columns loads one inside.
// `put` zeroes what is past `len` rows and `cols` columns. Fewer than 8 columns may be left of rows
// that hold 8 at least: the load then begins before them. Offsets are 32 bits of bytes, without a
// sign, from a base that is the same for all lanes, 8 elements before the tile: the least of them is
// one element (rows lie at least 0 and less than 2^24 elements apart).
template <typename T, int C, int W, int NT>
struct TileFetch {
  static constexpr int PER = C * W / 8, N = (PER + NT - 1) / NT;
  static constexpr uint32_t ES = sizeof(T);
  Piece<T> r[N];
  __device__ __forceinline__ static int row_of(int i, int tid) { return (i * NT + tid) / (W / 8); }
  __device__ __forceinline__ static int col_of(int i, int tid) {
    return (i * NT + tid) % (W / 8) * 8;
  }
  __device__ __forceinline__ void get(const T* src, long st, int len, int cols, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      r[i].get(src - 8, (uint32_t)min(row_of(i, tid), len - 1) * (uint32_t)st * ES +
                            (uint32_t)(min(col_of(i, tid), cols - 8) + 8) * ES);
  }
  // Whether a piece of the thread has a value that is not finite (one past the tile's rows or columns
  // says what the one that was loaded in its place says).
  __device__ __forceinline__ bool not_finite() const {
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) s |= r[i].full();
    return s & Piece<T>::SIGNS;
  }
  // The piece as it belongs into the tile.
  __device__ __forceinline__ Frag<T> piece(int i, int len, int cols, int tid) const {
    Frag<T> f = cut_frag<T>(r[i].frag(), col_of(i, tid), cols);
    return row_of(i, tid) < min(len, C) ? f : Frag<T>{};
  }
  __device__ __forceinline__ void put(T* dst, int pitch, int len, int cols, int tid) const {
    dst += row_of(0, tid) * pitch + col_of(0, tid);   // NT / (W / 8) rows from piece to piece
    constexpr int ROWS = NT / (W / 8);
    static_assert(NT % (W / 8) == 0, "the pieces of a thread lie in one column");
    if (PER % NT == 0 && len >= C && cols >= W) {
#pragma unroll
      for (int i = 0; i < N; ++i) st_frag(dst + i * ROWS * pitch, r[i].frag());
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (PER % NT == 0 || i * NT + tid < PER)
        st_frag(dst + i * ROWS * pitch, piece(i, len, cols, tid));
  }
};
// The same for tile after tile of one source, whose rows lie `st` >= 0 apart: their offsets stay in
// registers.
template <typename T, int C, int W, int NT>
struct TileStream : TileFetch<T, C, W, NT> {
  using Base = TileFetch<T, C, W, NT>;
  static_assert(NT % (W / 8) == 0, "the pieces of a thread lie in one column");
  uint32_t row[Base::N], col;
  __device__ __forceinline__ TileStream(long st, int cols, int tid)
      : col((uint32_t)(min(Base::col_of(0, tid), cols - 8) + 8) * Base::ES) {
#pragma unroll
    for (int i = 0; i < Base::N; ++i)
      row[i] = (uint32_t)Base::row_of(i, tid) * (uint32_t)st * Base::ES;
  }
  __device__ __forceinline__ void next(const T* src, int st, int len) {
    const uint32_t last = (uint32_t)(min(len, C) - 1) * (uint32_t)st * Base::ES;
#pragma unroll
    for (int i = 0; i < Base::N; ++i) Base::r[i].get(src - 8, min(row[i], last) + col);
  }
};
// [ROWS][32] tiles in a row, whole and aligned.
template <typename T, int ROWS, int NT>
struct BlockStream {
  static constexpr int PER = ROWS * 4, N = (PER + NT - 1) / NT;
  Frag<T> r[N];
  __device__ __forceinline__ void next(const T* src, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      r[i] = ld_frag(src + 8 * (PER % NT == 0 ? i * NT + tid : min(i * NT + tid, PER - 1)));
  }
  __device__ __forceinline__ void put(T* dst, int pitch, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i * NT + tid;
      if (PER % NT == 0 || p < PER) st_frag(dst + p / 4 * pitch + p % 4 * 8, r[i]);
    }
  }
};

// acc[i] += A(i) B for N tiles of rows, part after part of a split operand, so that a product does
// not wait for the one before it.
template <typename T, int N, int P, typename F>
__device__ __forceinline__ void mma_rows(f32x4 (&acc)[N], const F& rows, const Split<T, P>& b) {
  constexpr int W = N < 4 ? N : 4;
#pragma unroll
  for (int i = 0; i < N; i += W) {
    Frag<T> a[W];
#pragma unroll
    for (int x = 0; x < W; ++x) a[x] = rows(i + x);
#pragma unroll
    for (int part = P - 1; part >= 0; --part)
#pragma unroll
      for (int x = 0; x < W; ++x) mma(acc[i + x], a[x], b.p[part]);
  }
}
// The same with the rows in as many parts, for the pair of tiles u.
template <typename T, int N, int P, typename F>
__device__ __forceinline__ void mma_split_pair(f32x4 (&acc)[N], int u, const F& rows,
                                               const Split<T, P>& b) {
  const Split<T, P> a[2] = {rows(0), rows(1)};
#pragma unroll
  for (int s = P - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) mma(acc[2 * u + h], a[h].p[i], b.p[s - i]);
}

// A lane's rows of its column of a state: row k + 32 s + 4 h + r in S[2 s + h][r], k its first. `at`
// is the column in row 0. Rows past K are the last one's when they are loaded.
template <int N>
__device__ __forceinline__ void load_rows(f32x4 (&S)[N], const float* at, int k, int K, int V) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[i][r] = at[(long)min(k + 32 * (i >> 1) + 4 * (i & 1) + r, K - 1) * V];
}
template <int N>
__device__ __forceinline__ void store_rows(const f32x4 (&S)[N], float* at, int k, int K, int V) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = k + 32 * (i >> 1) + 4 * (i & 1) + r;
      if (row < K) at[(long)row * V] = S[i][r];
    }
}
// The same of all rows of a state for a wave's 16 columns, zeros where a lane has no column;
// `at` is then one inside.
template <int N>
__device__ __forceinline__ void load_state(f32x4 (&S)[N], const float* at, bool inside, int g,
                                           int K, int V) {
  load_rows(S, at, 8 * g, K, V);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (!inside || 32 * (i >> 1) + 8 * g + 4 * (i & 1) + r >= K) S[i][r] = 0.f;
}
template <int N>
__device__ __forceinline__ void store_state(const f32x4 (&S)[N], float* at, bool inside, int g,
                                            int K, int V) {
  if (inside) store_rows(S, at, 8 * g, K, V);
}

}  // namespace tops
