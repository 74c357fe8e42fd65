// Layer norm and its gradients (include/tops_gla_delta.h).
//
//   y  = (x - mean) rstd w + b
//   dx = rstd (u - mean(u) - n mean(u n)),  u = dy w,  n = (x - mean) rstd,
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Bound by memory: x (and dy) are read once into registers, the mean comes before the squares of
// the differences (a variance from sum and sum of squares loses what a large mean covers), and the
// next row's loads are on their way while a row is worked on. A thread holds at most 16 features,
// whose share of w, b, dw and db stays in its registers over all its rows: up to 1024 features a row
// belongs to one wave, above to a block of 2 to 16. The weights' sums go through one partial row a
// block in a workspace and a second kernel, in fixed order.
//
// What bounds it is how many loads are on their way: the gradients of 32768 x 2048 bfloat16, 403 MB,
// take 84 us, 4.8 TB/s, with 8 features a thread and 20 waves a CU, with 16 features, twice the
// registers, and 12 waves 105, 8 waves 139. In float32 16 features are as many bytes again: 16384 x
// 2048 in 91 us, sums included, with 8 waves of 16 features, 95 with 20 of 8; 65536 x 768 in 123 with
// 8 waves, 128 with 12. The forward's 268 MB take 64 us, 4.2 TB/s, with 16 features (with 8: 71). The
// sums over 1280 blocks' partial rows take 5 with 8 of a thread's loads on their way, 12 with one.
#include "delta.hpp"

namespace tops {

namespace {

// Threads of a row by its features: 16 a thread, or 8 (`few`: the gradients of bfloat16), but 16 where
// 64 threads have them (a block of 128 would write a partial row for each row) or 1024 threads must.
// And of a block: four rows of one wave, or one row.
int row_threads(long D, bool few) {
  if (D <= 1024) return 64;
  const long n = few ? D : D / 2 + D % 2;
  return n <= 1024 ? 128 : n <= 2048 ? 256 : n <= 4096 ? 512 : 1024;
}
constexpr int block_threads(int nt) { return nt == 64 ? 256 : nt; }
// The blocks that run at once, in whole ones a CU (few features leave registers for 20 waves, 16 of
// them in bfloat16 for 12).
long norm_blocks(long rows, long D, bool backward, bool bf16) {
  const int nt = row_threads(D, backward && bf16), bt = block_threads(nt);
  const long per = bt / nt, waves = !backward ? 16 : !bf16 ? 8 : D <= 8 * nt ? 20 : 12;
  const long most = std::max(1L, waves * 64 / bt) * 256;
  return std::min((rows + per - 1) / per, most);
}

__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0x121>(x);
  x += dpp<0x122>(x);
  x += dpp<0x124>(x);
  x += dpp<0x128>(x);
  x = swap16_add(x, x);
  return swap32_add(x, x);
}
// Sums of N values over the threads of a row; `sm` is one of two places that take turns, so that a
// sum needs one barrier.
template <int NT, int N>
__device__ __forceinline__ void row_sum(float (&x)[N], float (*sm)[16], int tid) {
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = wave_sum(x[n]);
  if constexpr (NT > 64) {
    if ((tid & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) sm[n][tid >> 6] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[n] = 0.f;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) x[n] += sm[n][i];
    }
  }
}

// Features c .. c + VEC - 1 of run i of a thread: runs of a row's threads lie side by side.
template <int NT, int VEC>
__device__ __forceinline__ int run_col(int tid, int i) {
  return (i * NT + tid) * VEC;
}

// The VEC features from c on of a row of D, zeros past its end. Where VEC divides D the load has no
// condition (a run past the end loads the last one), so that a row's loads are all on their way at
// once; the caller leaves such a run out.
template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> load_run(const T* row, int c, int D) {
  if (D % VEC == 0) return get_run<T, VEC>(row + min(c, D - VEC));
  Run<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = c + e < D ? row[c + e] : zero_elem<T>();
  return r;
}

template <int NT, int R, int VEC>
__device__ __forceinline__ void load_weights(const float* w, int D, int tid, float none,
                                             float (&x)[R][VEC]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int c = run_col<NT, VEC>(tid, i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[i][e] = none;
    if (w) {
      const auto r = load_run<float, VEC>(w, c, D);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[i][e] = c + e < D ? r.v[e] : 0.f;
    }
  }
}

template <typename T, int NT, int R>
__global__ __launch_bounds__(block_threads(NT)) void layer_norm_fwd_kernel(
    tops_gla_layer_norm_args a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int PER = block_threads(NT) / NT;
  __shared__ float sm[2][1][16];
  const int D = (int)a.D, tid = threadIdx.x % NT;
  const float eps = (float)a.eps;
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  float w[R][VEC], b[R][VEC];
  load_weights<NT, R, VEC>(a.w, D, tid, 1.f, w);
  load_weights<NT, R, VEC>(a.b, D, tid, 0.f, b);
  const long step = (long)gridDim.x * PER;
  long row = (long)blockIdx.x * PER + threadIdx.x / NT;
  Run<T, VEC> nx[R];
  auto load = [&](long r) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      nx[i] = load_run<T, VEC>(x + r * a.x_st, run_col<NT, VEC>(tid, i), D);
    }
  };
  if (row < a.rows) load(row);
  for (; row < a.rows; row += step) {
    float v[R][VEC], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool in = run_col<NT, VEC>(tid, i) < D;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = in ? to_f32(nx[i].v[e]) : 0.f;
        s[0] += v[i][e];
      }
    }
    if (row + step < a.rows) load(row + step);
    row_sum<NT>(s, sm[0], tid);
    const float mean = s[0] / (float)D;   // a row of one value has exactly its mean
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = c + e < D ? v[i][e] - mean : 0.f;
        s[0] = fmaf(v[i][e], v[i][e], s[0]);
      }
    }
    row_sum<NT>(s, sm[1], tid);
    const float rstd = 1.f / sqrtf(s[0] / (float)D + eps);
    if (a.stats && tid == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
      float r[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] = fmaf(v[i][e] * rstd, w[i][e], b[i][e]);
      if (c < D) put_run<T, VEC>(y + row * D + c, r, D - c);
    }
  }
}

template <typename T, int NT, int R>
__global__ __launch_bounds__(block_threads(NT)) void layer_norm_bwd_kernel(
    tops_gla_layer_norm_args a) {
  constexpr int VEC = 16 / (int)sizeof(T), PER = block_threads(NT) / NT;
  __shared__ float sm[2][2][16];
  __shared__ float part[PER > 1 ? 2 * R * VEC * NT : 1];
  const int D = (int)a.D, tid = threadIdx.x % NT;
  const T *x = (const T*)a.x, *dy = (const T*)a.dy;
  T* dx = (T*)a.dx;
  float w[R][VEC], dw[R][VEC], db[R][VEC];
  load_weights<NT, R, VEC>(a.w, D, tid, 1.f, w);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
  const long step = (long)gridDim.x * PER;
  long row = (long)blockIdx.x * PER + threadIdx.x / NT;
  Run<T, VEC> nx[R], nd[R];
  float mean = 0.f, rstd = 0.f;
  const float inv = 1.f / (float)D;
  int turn = 0;
  auto load = [&](long r) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
      nx[i] = load_run<T, VEC>(x + r * a.x_st, c, D);
      nd[i] = load_run<T, VEC>(dy + r * a.dy_st, c, D);
    }
    mean = a.stats[2 * r];
    rstd = a.stats[2 * r + 1];
  };
  if (row < a.rows) load(row);
  for (; row < a.rows; row += step) {
    float n[R][VEC], u[R][VEC], s[2] = {0.f, 0.f};
    const float m = mean, rs = rstd;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool in = c + e < D;
        n[i][e] = in ? (to_f32(nx[i].v[e]) - m) * rs : 0.f;
        const float d = in ? to_f32(nd[i].v[e]) : 0.f;
        db[i][e] += d;
        dw[i][e] = fmaf(d, n[i][e], dw[i][e]);
        u[i][e] = d * w[i][e];
        s[0] += u[i][e];
        s[1] = fmaf(u[i][e], n[i][e], s[1]);
      }
    }
    if (row + step < a.rows) load(row + step);
    row_sum<NT>(s, sm[turn], tid);
    turn ^= 1;
    const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
      float r[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] = rs * (u[i][e] - m1 - n[i][e] * m2);
      if (c < D) put_run<T, VEC>(dx + row * D + c, r, D - c);
    }
  }
  if (!a.ws) return;
  float* out = (float*)a.ws + (long)blockIdx.x * 2 * D;
  if constexpr (PER > 1) {   // the block's waves one after another, in their order
    for (int p = 0; p < PER; ++p) {
      if ((int)threadIdx.x / NT == p) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float* q = part + (i * VEC + e) * NT + tid;
            q[0] = p ? q[0] + dw[i][e] : dw[i][e];
            q[R * VEC * NT] = p ? q[R * VEC * NT] + db[i][e] : db[i][e];
          }
      }
      __syncthreads();
    }
    if ((int)threadIdx.x < NT) {
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dw[i][e] = part[(i * VEC + e) * NT + tid];
          db[i][e] = part[(R * VEC + i * VEC + e) * NT + tid];
        }
    }
  }
  if ((int)threadIdx.x < NT) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = run_col<NT, VEC>(tid, i);
      if (c < D) {
        put_run<float, VEC>(out + c, dw[i], D - c);
        put_run<float, VEC>(out + D + c, db[i], D - c);
      }
    }
  }
}

// Sums `parts` rows of 2 D partial sums: 32 columns a block, a thirty-second of the rows for each
// half of its waves.
__global__ __launch_bounds__(1024) void layer_norm_sum_kernel(const float* ws, int parts, int D,
                                                              float* dw, float* db) {
  __shared__ float sm[32][33];
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int r = part; r < parts; r += 32) s += ws[(long)r * 2 * D + c];
  }
  sm[part][col] = s;
  __syncthreads();
  if (part == 0 && c < 2 * D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sm[i][col];
    if (c < D) {
      if (dw) dw[c] = s;
    } else if (db) {
      db[c - D] = s;
    }
  }
}

template <typename T, int NT, int R, bool BACK>
void launch(const tops_gla_layer_norm_args& a, hipStream_t st) {
  const int nb = (int)norm_blocks(a.rows, a.D, BACK, sizeof(T) == 2);
  if constexpr (BACK)
    layer_norm_bwd_kernel<T, NT, R><<<nb, block_threads(NT), 0, st>>>(a);
  else
    layer_norm_fwd_kernel<T, NT, R><<<nb, block_threads(NT), 0, st>>>(a);
}
// The runs of a thread: rows of more than a wave are more than half of what their threads hold.
template <typename T, int NT, bool BACK>
void launch(const tops_gla_layer_norm_args& a, hipStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T), MOST = 16 / VEC;
  constexpr bool FEW = BACK && sizeof(T) == 2;
  if constexpr (NT == 64) {
    if (a.D <= 64 * VEC) return launch<T, NT, 1, BACK>(a, st);
    if (VEC == 4 && a.D <= 128 * VEC) return launch<T, NT, 2, BACK>(a, st);
    launch<T, NT, MOST, BACK>(a, st);
  } else if constexpr (!FEW) {
    launch<T, NT, MOST, BACK>(a, st);
  } else {
    if (NT < 1024 || a.D <= 8 * NT) return launch<T, NT, MOST / 2, BACK>(a, st);
    if constexpr (NT == 1024) launch<T, NT, MOST, BACK>(a, st);
  }
}

template <typename T, bool BACK>
hipError_t run(const tops_gla_layer_norm_args& a, hipStream_t st) {
  if (a.rows > 0) {
    constexpr bool FEW = BACK && sizeof(T) == 2;
    switch (row_threads(a.D, FEW)) {
      case 64: launch<T, 64, BACK>(a, st); break;
      case 128:
        if constexpr (!FEW) launch<T, 128, BACK>(a, st);
        break;
      case 256: launch<T, 256, BACK>(a, st); break;
      case 512: launch<T, 512, BACK>(a, st); break;
      default: launch<T, 1024, BACK>(a, st);
    }
  }
  if (BACK && a.ws) {
    const int parts = (int)norm_blocks(a.rows, a.D, true, sizeof(T) == 2);
    layer_norm_sum_kernel<<<(unsigned)((2 * a.D + 31) / 32), 1024, 0, st>>>(
        (const float*)a.ws, parts, (int)a.D, a.dw, a.db);
  }
  return hipGetLastError();
}

}  // namespace

long layer_norm_part_rows(long rows, long D, int dtype) {
  return norm_blocks(rows, D, true, dtype == DT_BF16);
}

hipError_t run_layer_norm_fwd(const tops_gla_layer_norm_args& a, hipStream_t st) {
  return a.dtype == DT_BF16 ? run<bf16, false>(a, st) : run<float, false>(a, st);
}
hipError_t run_layer_norm_bwd(const tops_gla_layer_norm_args& a, hipStream_t st) {
  return a.dtype == DT_BF16 ? run<bf16, true>(a, st) : run<float, true>(a, st);
}

}  // namespace tops
