// socmx_layernorm.hip -- layer norm over the last dimension, forward and backward, gfx950.
//
//   mu = mean_j x_j,  s2 = mean_j (x_j - mu)^2,  r = 1 / sqrt(s2 + eps),  n_j = (x_j - mu) r,  y_j = n_j w_j + b_j
//   dx_j = r (g_j - mean(g) - n_j mean(g n)),  g = dy w;     dw_j = sum_rows dy_j n_j,   db_j = sum_rows dy_j
//
// Both directions are bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx.  A row
// is read ONCE into the registers of the L lanes that own it (at most 16 elements a lane), the variance is the sum of squared
// differences from the mean (no cancellation of large squares), and the mean of those differences -- what rounding left of the mean,
// times 1 / sqrt(eps) an error of its own where a row hardly varies -- is taken off once more with the same reduction; all statistics
// are f32.  The mean that is kept for the backward is one f32, which does not hold that rest: there n = (x - mean) r has a mean c of its own,
// formed beside the other two sums of a row and taken off, n - c (and mean(g n) - c mean(g)).  L is a power of two: several short
// rows share a wave, rows of more than 1024 elements take L / 64 waves that meet in LDS.  In the backward every lane keeps
// the weight and bias gradients of its columns over all the rows its workgroup takes; the workgroup's sums go to a slot of
// their own and a second launch adds the slots in a fixed order: no atomics, the same bits on every run.  Rows of more than
// 16384 elements are read again from the caches instead of being kept (the *_long kernels).
//
// MEASURED.  bf16 (8192, 4096): forward 27.5 us (4.9 TB/s), backward 41.5 (4.9; 40 without the sum of n) and 4 for the slots, a copy of this size runs
// at 5.3 to 6.8; f32 (25728, 256): 11 (4.8), 16.5 (4.8) and 3.6; f32 (4096, 12288): 91 (4.4), 105 (5.8) and 6.  f16 (4111, 1601), y, dy and dx at odd
// addresses: 12, 17 and 5.5, a third of that rate: one row a workgroup at a time, so what is left is the way of one row through its sums, and
// in the backward the slots.  y leaves past the caches (28.5 -> 26.5 us); dx did not gain.  The first shape's forward with 8 elements a lane
// (twice the waves a row) 30 us, with 32 28, alone 24.6; (4111, 1601) 11.0, 13.6 and 10.8.  bf16 (512, 50000): 34, 42, 21.5 and 10.6.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/socmx.h"
#include "socmx_launch.h"
#include "socmx_vec.h"

namespace socmx {

struct NormArgs {
  const void *x, *dy, *w, *b;        // w, b nullable; their type: f32 when w32, else x's
  void *y, *dx, *dw, *db;            // y of the forward; dx, dw, db of the backward, each nullable
  float *mean, *rstd;                // (rows,); nullable together in the forward
  float* part;                       // backward: (slots, 2, cols)
  float* shift;                      // backward of long rows: (rows,), the c of every row (with part only)
  int64_t rows, x_stride, dy_stride; // elements between rows; y and dx are dense
  int cols, w32;
  float eps;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(float (&out)[VEC], const void* w, int w32, int col, int cols, float missing) {
  const int n = cols - col;
  if (!w || n <= 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = missing;
  } else if (w32) {
    const reg_vec<float, VEC> v = load_vec<float, VEC>(static_cast<const float*>(w) + col, n);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = v[i];
  } else {
    const reg_vec<T, VEC> v = load_vec<T, VEC>(static_cast<const T*>(w) + col, n);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = v[i];
  }
}

// totals of N sums over the L lanes (L / 64 waves) of a row; `red`: N L / 64 floats, free again after the next call's barrier
template <int L, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* red) {
  constexpr int W = L <= 64 ? 1 : L / 64;
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = lanes_sum<(L <= 64 ? L : 64)>(s[k]);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) red[k * W + (threadIdx.x >> 6)] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) s[k] += red[k * W + i];
    }
  }
}

template <typename T, int VEC, int NV, int L>
__global__ __launch_bounds__(L <= 64 ? 256 : L) void layer_norm_fwd_kernel(const NormArgs a) {
  constexpr int THREADS = L <= 64 ? 256 : L, GROUPS = THREADS / L;
  __shared__ float red[2][2 * (L <= 64 ? 1 : L / 64)];
  const int lane = threadIdx.x % L;
  const int64_t first = (int64_t)blockIdx.x * GROUPS + threadIdx.x / L, stride = (int64_t)gridDim.x * GROUPS;
  const float cols = (float)a.cols;
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_weight<T, VEC>(w[v], a.w, a.w32, (v * L + lane) * VEC, a.cols, 1.f);
    load_weight<T, VEC>(b[v], a.b, a.w32, (v * L + lane) * VEC, a.cols, 0.f);
  }
  for (int64_t row = first; row < a.rows; row += stride) {      // (L > 64: the same rows for the whole workgroup)
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float e[NV][VEC], s[1] = {}, d[2] = {};              // sums of x; of x - mean and of its square
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * L + lane) * VEC;
      reg_vec<T, VEC> raw = load_vec<T, VEC>(x + (col < a.cols ? col : 0), col < a.cols ? a.cols - col : 0);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += e[v][i] = raw[i];
    }
    row_sums<L>(s, red[0]);
    const float mean = s[0] / cols;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        e[v][i] -= mean;
        if ((v * L + lane) * VEC + i < a.cols) {
          d[0] += e[v][i];
          d[1] += e[v][i] * e[v][i];
        }
      }
    row_sums<L>(d, red[1]);
    const float rest = d[0] / cols, var = d[1] / cols - rest * rest, r = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * L + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[v][i] = (e[v][i] - rest) * r * w[v][i] + b[v][i];
      if (col < a.cols) stream_vec<T, VEC>(y + col, e[v], a.cols - col);
    }
    if (a.mean && lane == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = r;
    }
  }
}

// n here is (x - mean) r, its mean c is known after a row's sums: dx has c in what is the same for the whole row, dw gets its share then.
// WEIGHTS: the gradients of weight and bias are wanted.  Which operations are fused is written down, so that a gradient has the same bits
// whichever others are wanted with it.
template <typename T, int VEC, int NV, int L, bool WEIGHTS>
__global__ __launch_bounds__(L <= 64 ? 256 : L) void layer_norm_bwd_kernel(const NormArgs a) {
#pragma clang fp contract(off)
  constexpr int THREADS = L <= 64 ? 256 : L, GROUPS = THREADS / L, WAVES = THREADS / 64;
  __shared__ float red[2][3 * (L <= 64 ? 1 : L / 64)];
  const int lane = threadIdx.x % L;
  const int64_t first = (int64_t)blockIdx.x * GROUPS + threadIdx.x / L, stride = (int64_t)gridDim.x * GROUPS;
  const float inv = 1.f / (float)a.cols;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_weight<T, VEC>(w[v], a.w, a.w32, (v * L + lane) * VEC, a.cols, 1.f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[v][i] = db[v][i] = 0.f;
  }
  int turn = 0;
  for (int64_t row = first; row < a.rows; row += stride, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], r = a.rstd[row];
    float n[NV][VEC], sum[3] = {};                       // sums of g, of g n and of n
    reg_vec<T, VEC> rd[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * L + lane) * VEC;
      const int have = col < a.cols ? a.cols - col : 0;
      const reg_vec<T, VEC> rx = load_vec<T, VEC>(x + (have ? col : 0), have);
      rd[v] = load_vec<T, VEC>(dy + (have ? col : 0), have);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {               // (behind the row's end dy = 0: what has it for a factor is 0)
        n[v][i] = (rx[i] - mean) * r;
        if constexpr (WEIGHTS) {
          dw[v][i] = fmaf(rd[v][i], n[v][i], dw[v][i]);
          db[v][i] += rd[v][i];
        }
        const float g = rd[v][i] * w[v][i];
        sum[0] += g;
        sum[1] = fmaf(g, n[v][i], sum[1]);
        sum[2] += i < have ? n[v][i] : 0.f;
      }
    }
    row_sums<L>(sum, red[turn]);
    const float s = sum[0] * inv, c = sum[2] * inv, q = fmaf(-c, s, sum[1] * inv), both = fmaf(-c, q, s);
    T* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * L + lane) * VEC;
      float e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (WEIGHTS) dw[v][i] = fmaf(-c, rd[v][i], dw[v][i]);
        e[i] = r * fmaf(-n[v][i], q, fmaf(rd[v][i], w[v][i], -both));
      }
      if (a.dx && col < a.cols) store_vec<T, VEC>(dx + col, e, a.cols - col);
    }
  }
  if constexpr (WEIGHTS) {
    float* slot = a.part + (int64_t)blockIdx.x * 2 * a.cols;
    if constexpr (L > 64) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = (v * L + lane) * VEC;
        if (col < a.cols) {
          store_vec<float, VEC>(slot + col, dw[v], a.cols - col);
          store_vec<float, VEC>(slot + a.cols + col, db[v], a.cols - col);
        }
      }
    } else {
      // the groups of a wave, then the waves
      __shared__ float acc[WAVES][2][L * NV * VEC];
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
#pragma unroll
          for (int off = L; off < 64; off *= 2) {
            dw[v][i] += __shfl_xor(dw[v][i], off, 64);
            db[v][i] += __shfl_xor(db[v][i], off, 64);
          }
          if ((threadIdx.x & 63) < L) {
            acc[threadIdx.x >> 6][0][(v * L + lane) * VEC + i] = dw[v][i];
            acc[threadIdx.x >> 6][1][(v * L + lane) * VEC + i] = db[v][i];
          }
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += THREADS) {
        float sw = 0.f, sb = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
          sw += acc[k][0][c];
          sb += acc[k][1][c];
        }
        slot[c] = sw;
        slot[a.cols + c] = sb;
      }
    }
  }
}

// ---- rows that do not fit the registers: 1024 threads a row, the row read again for each sum ---------------------------------
template <typename T, int VEC>
__global__ __launch_bounds__(1024) void layer_norm_fwd_long_kernel(const NormArgs a) {
  __shared__ float red[2][32];
  const float cols = (float)a.cols;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float s[1] = {}, d[2] = {};
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      const reg_vec<T, VEC> v = load_vec<T, VEC>(x + col, a.cols - col);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[i];
    }
    row_sums<1024>(s, red[0]);
    const float mean = s[0] / cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      const reg_vec<T, VEC> v = load_vec<T, VEC>(x + col, a.cols - col);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col + i < a.cols) {
          d[0] += v[i] - mean;
          d[1] += (v[i] - mean) * (v[i] - mean);
        }
    }
    row_sums<1024>(d, red[1]);
    const float rest = d[0] / cols, var = d[1] / cols - rest * rest, r = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      const reg_vec<T, VEC> v = load_vec<T, VEC>(x + col, a.cols - col);
      float w[VEC], b[VEC], e[VEC];
      load_weight<T, VEC>(w, a.w, a.w32, col, a.cols, 1.f);
      load_weight<T, VEC>(b, a.b, a.w32, col, a.cols, 0.f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = ((v[i] - mean) - rest) * r * w[i] + b[i];
      stream_vec<T, VEC>(y + col, e, a.cols - col);
    }
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = r;
    }
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(1024) void layer_norm_bwd_long_kernel(const NormArgs a) {
  __shared__ float red[2][48];
  const float inv = 1.f / (float)a.cols;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], r = a.rstd[row];
    float sum[3] = {}, w[VEC], e[VEC];
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      const reg_vec<T, VEC> vx = load_vec<T, VEC>(x + col, a.cols - col), vd = load_vec<T, VEC>(dy + col, a.cols - col);
      load_weight<T, VEC>(w, a.w, a.w32, col, a.cols, 1.f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float n = (vx[i] - mean) * r, g = vd[i] * w[i];
        sum[0] += g;
        sum[1] += g * n;
        sum[2] += i < a.cols - col ? n : 0.f;
      }
    }
    row_sums<1024>(sum, red[turn]);
    const float s = sum[0] * inv, c = sum[2] * inv, q = sum[1] * inv - c * s;
    if (a.shift && threadIdx.x == 0) a.shift[row] = c;
    if (!a.dx) continue;
    T* dx = static_cast<T*>(a.dx) + row * a.cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += 1024 * VEC) {
      const reg_vec<T, VEC> vx = load_vec<T, VEC>(x + col, a.cols - col), vd = load_vec<T, VEC>(dy + col, a.cols - col);
      load_weight<T, VEC>(w, a.w, a.w32, col, a.cols, 1.f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = r * (vd[i] * w[i] - s - ((vx[i] - mean) * r - c) * q);
      store_vec<T, VEC>(dx + col, e, a.cols - col);
    }
  }
}

// long rows' weight gradients: a workgroup takes 256 VEC columns and every gridDim.y-th row
template <typename T, int VEC>
__global__ __launch_bounds__(256) void layer_norm_bwd_long_weights_kernel(const NormArgs a) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * VEC;
  if (col >= a.cols) return;
  float dw[VEC], db[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) dw[i] = db[i] = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const reg_vec<T, VEC> vx = load_vec<T, VEC>(static_cast<const T*>(a.x) + row * a.x_stride + col, a.cols - col);
    const reg_vec<T, VEC> vd = load_vec<T, VEC>(static_cast<const T*>(a.dy) + row * a.dy_stride + col, a.cols - col);
    const float mean = a.mean[row], r = a.rstd[row], c = a.shift[row];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      dw[i] += vd[i] * ((vx[i] - mean) * r - c);
      db[i] += vd[i];
    }
  }
  float* slot = a.part + (int64_t)blockIdx.y * 2 * a.cols;
  store_vec<float, VEC>(slot + col, dw, a.cols - col);
  store_vec<float, VEC>(slot + a.cols + col, db, a.cols - col);
}

// adds the workgroups' slots: 32 columns a workgroup, 32 strands over the slots, joined in order (8 strands: 9 us for 5
// with 1024 slots of 2 x 1601)
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_bwd_finish_kernel(const float* __restrict__ part, int slots, int cols,
                                                                    T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float red[32][32];
  const int k = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + k;
  float s = 0.f;
  if (c < 2 * (int64_t)cols) {
#pragma unroll 8
    for (int i = strand; i < slots; i += 32) s += part[(int64_t)i * 2 * cols + c];
  }
  red[strand][k] = s;
  __syncthreads();
  if (strand == 0 && c < 2 * (int64_t)cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += red[i][k];
    if (c < cols) {
      if (dw) dw[c] = (T)s;
    } else if (db) {
      db[c - cols] = (T)s;
    }
  }
}

// ---- which kernel: 16 elements a lane at most, the fewest lanes that hold the row ---------------------------------------------
static const int kNormKept = 16384;

static inline int norm_lanes(int cols, int vec) {
  const int vectors = (cols + vec - 1) / vec;
  if (vectors <= 64) {
    int lanes = 8;
    while (lanes < vectors) lanes *= 2;
    return lanes;
  }
  int lanes = 64;
  while (lanes * 16 < cols) lanes *= 2;
  return lanes;
}

// the backward's workgroups, each with a slot of weight gradients: eight waves for every CU at most (a workgroup for every CU at least).  What the
// slots add to the rows' traffic, written and read: 3 % for (25728, 256) f32, 17 % for (8192, 4096) bf16, 66 % for (4111, 1601) f16, 4 rows a slot
static inline int64_t norm_slots(int64_t rows, int cols, int vec) {
  if (cols > kNormKept) return std::min<int64_t>(rows, 64);
  const int lanes = norm_lanes(cols, vec), groups = lanes <= 64 ? 256 / lanes : 1;
  const int64_t most = lanes <= 64 ? 512 : std::max(256, 512 * 256 / lanes);
  return std::max<int64_t>(1, std::min<int64_t>(most, (rows + groups - 1) / groups));
}

template <typename T, bool BWD, int VEC, int NV, int L>
static int launch_norm_kernel(const NormArgs& a, int64_t blocks, void* stream) {
  const dim3 block(L <= 64 ? 256 : L);
  if constexpr (!BWD)
    return launch(layer_norm_fwd_kernel<T, VEC, NV, L>, dim3((unsigned)blocks), block, 0, stream, a);
  else if (a.part)
    return launch(layer_norm_bwd_kernel<T, VEC, NV, L, true>, dim3((unsigned)blocks), block, 0, stream, a);
  else
    return launch(layer_norm_bwd_kernel<T, VEC, NV, L, false>, dim3((unsigned)blocks), block, 0, stream, a);
}

template <typename T, bool BWD>
static int launch_norm(const NormArgs& a, int64_t slots, void* stream) {
  constexpr int VEC = 16 / sizeof(T);
  if (a.cols > kNormKept) {
    const unsigned blocks = (unsigned)std::min<int64_t>(a.rows, 1024);
    if constexpr (!BWD) return launch(layer_norm_fwd_long_kernel<T, VEC>, dim3(blocks), dim3(1024), 0, stream, a);
    int err = launch(layer_norm_bwd_long_kernel<T, VEC>, dim3(blocks), dim3(1024), 0, stream, a);
    if (err == 0 && a.part)
      err = launch(layer_norm_bwd_long_weights_kernel<T, VEC>, dim3((unsigned)((a.cols + 256 * VEC - 1) / (256 * VEC)), (unsigned)slots),
                   dim3(256), 0, stream, a);
    return err;
  }
  const int lanes = norm_lanes(a.cols, VEC), per_lane = (a.cols + lanes * VEC - 1) / (lanes * VEC);
  const int groups = lanes <= 64 ? 256 / lanes : 1;
  const int64_t blocks = BWD && a.part ? slots : std::min<int64_t>((a.rows + groups - 1) / groups, lanes <= 64 ? 2048 : 2048 * 256 / lanes);
#define SOCMX_NORM(LANES, N) return launch_norm_kernel<T, BWD, VEC, N, LANES>(a, blocks, stream)
  constexpr int FULL = 16 / VEC;
  switch (lanes) {
    case 8: SOCMX_NORM(8, 1);
    case 16: SOCMX_NORM(16, 1);
    case 32: SOCMX_NORM(32, 1);
    case 64:
      if (per_lane == 1) SOCMX_NORM(64, 1);
      if (per_lane == 2) SOCMX_NORM(64, 2);
      SOCMX_NORM(64, FULL);
    case 128: SOCMX_NORM(128, FULL);
    case 256: SOCMX_NORM(256, FULL);
    case 512: SOCMX_NORM(512, FULL);
    default: SOCMX_NORM(1024, FULL);
  }
#undef SOCMX_NORM
}

template <bool BWD>
static int dispatch_norm(int32_t type, const NormArgs& a, int64_t slots, void* stream) {
  if (type == SOCMX_F32) return launch_norm<float, BWD>(a, slots, stream);
  if (type == SOCMX_BF16) return launch_norm<bf16_t, BWD>(a, slots, stream);
  return launch_norm<f16_t, BWD>(a, slots, stream);
}

static inline int norm_check(int32_t type, int32_t wtype, int64_t rows, int64_t cols) {
  if (type < SOCMX_F32 || type > SOCMX_F16 || (wtype != type && wtype != SOCMX_F32)) return SOCMX_E_KIND;
  if (rows < 1 || cols < 1 || cols > (1 << 24)) return SOCMX_E_DIM;
  return 0;
}

}  // namespace socmx

using namespace socmx;

extern "C" int socmx_layer_norm_fwd(int32_t type, int32_t wtype, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
                                    const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                                    socmx_stream_t stream) {
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return SOCMX_E_NULL;
  if (const int bad = norm_check(type, wtype, rows, cols)) return bad;
  NormArgs a = {};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.cols = (int)cols; a.x_stride = x_stride; a.w32 = wtype == SOCMX_F32; a.eps = eps;
  return dispatch_norm<false>(type, a, 0, stream);
}

extern "C" int64_t socmx_layer_norm_bwd_workspace_floats(int32_t type, int64_t rows, int64_t cols) {
  if (norm_check(type, type, rows, cols)) return 0;
  // (long rows: a float for each of them behind the slots, in whole slots)
  const int64_t more = cols > kNormKept ? (rows + 2 * cols - 1) / (2 * cols) : 0;
  return (norm_slots(rows, (int)cols, type == SOCMX_F32 ? 4 : 8) + more) * 2 * cols;
}

extern "C" int socmx_layer_norm_bwd(int32_t type, int32_t wtype, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
                                    const void* dy, int64_t dy_stride, const void* weight, const float* mean, const float* rstd,
                                    void* dx, void* dweight, void* dbias, float* workspace, socmx_stream_t stream) {
  if (!x || !dy || !mean || !rstd || (!dx && !dweight && !dbias)) return SOCMX_E_NULL;
  if ((dweight || dbias) && !workspace) return SOCMX_E_WORKSPACE;
  if (const int bad = norm_check(type, wtype, rows, cols)) return bad;
  NormArgs a = {};
  a.x = x; a.dy = dy; a.w = weight; a.dx = dx; a.dw = dweight; a.db = dbias;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.part = dweight || dbias ? workspace : nullptr;
  a.rows = rows; a.cols = (int)cols; a.x_stride = x_stride; a.dy_stride = dy_stride; a.w32 = wtype == SOCMX_F32;
  const int64_t slots = norm_slots(rows, (int)cols, type == SOCMX_F32 ? 4 : 8);
  if (a.part && cols > kNormKept) a.shift = a.part + slots * 2 * cols;
  int err = dispatch_norm<true>(type, a, slots, stream);
  if (err || !a.part) return err;
  const dim3 grid((unsigned)((2 * cols + 31) / 32)), block(1024);
  if (wtype == SOCMX_F32)
    return launch(layer_norm_bwd_finish_kernel<float>, grid, block, 0, stream, workspace, (int)slots, (int)cols, (float*)dweight, (float*)dbias);
  if (wtype == SOCMX_BF16)
    return launch(layer_norm_bwd_finish_kernel<bf16_t>, grid, block, 0, stream, workspace, (int)slots, (int)cols, (bf16_t*)dweight, (bf16_t*)dbias);
  return launch(layer_norm_bwd_finish_kernel<f16_t>, grid, block, 0, stream, workspace, (int)slots, (int)cols, (f16_t*)dweight, (f16_t*)dbias);
}
