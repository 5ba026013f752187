// socmx_scan.hip -- the gated linear recurrence along a trajectory, forward, backward and one step, gfx950.
//
//   h_t = a_t h_{t-1} + x_t,   a_t = exp(alpha_t),   h_{-1} = initial          x, h (T, B, D);  alpha (T, B, G), a gate per D / G channels
//   G_t = dh_t + a_{t+1} G_{t+1}:   dx_t = G_t,   dalpha_t = a_t h_{t-1} G_t (summed over a gate's channels),   dinitial = a_0 G_0
// in either direction of time (`reverse`) and up to a length of its own for every row b (`lengths`): "step k" below is the row's
// k-th step in its direction, the steps behind its length leave the state alone and get zeros.
//
// THE GATE.  A memory of n steps has a = 1 - 1/n: rounding a to f32 moves the steady state x / (1 - a) by n 2^-25, the same way
// on every step of a constant decay.  So a gate near 1 (-1/4 < alpha <= 0) is kept as q = exp(alpha) - 1 (a polynomial, full relative
// precision) and applied as h + q h, any other as q = exp(alpha); the sign of q tells them apart, and q = +0 (exp flushes
// what is below 2^-126) is a gate that forgets: whatever stood before it, infinities and NaN included, is replaced, not multiplied.
//
// ONE PASS.  A step is an affine map, so a run of steps is one: h -> exp(S) h + l with S = the sum of alpha and l its result from
// zero -- the same form, so a run is applied with the code of a step.  A workgroup owns 64 V channels and walks time in tiles of
// W waves x U steps: every wave holds its U steps in registers, forms its run's (q, l), the waves exchange them in LDS behind ONE
// barrier, each then applies the runs in front of it and finishes its own steps.  x and alpha are read once, h is written once; the
// next tile's loads are in flight meanwhile.  Bound by memory.  The state at the start of every tile is kept for the backward
// (f32, 1 / (W U) of h).
//
// THE BACKWARD walks the tiles from the end, rebuilds the tile's h from that state in f32 -- h itself, rounded to 16 bits, would
// put its rounding into dalpha -- and runs the same scheme on G: x, alpha and dh are read once, dx and dalpha written once.  A gate
// shared by several channels: their products are summed across the lanes in a fixed order, gates wider than a wave leave one partial
// sum a wave for a second launch.  No atomics: the same bits on every run.
//
// FEW CHANNELS, LONG TIME: time is cut into chunks; a first launch forms every chunk's (S, l), the second one composes the chunks
// in front of its own and proceeds as above (x and alpha are read twice).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/socmx.h"
#include "socmx_launch.h"
#include "socmx_vec.h"

namespace socmx {

struct ScanArgs {
  const void *x, *alpha, *dh;        // dh nullable (zeros)
  void *h, *dx, *dalpha;
  const float *initial, *dfinal;     // (B, D), nullable (zeros)
  float *final, *dinitial;           // (B, D), nullable
  float* state;                      // (tiles, B D): the state at the start of every tile; written by the forward when not NULL
  float* run;                        // (chunks, 2, B D): S and l of every chunk (more than one chunk only)
  float* part;                       // (T, B G, segments): partial sums of dalpha (gates wider than a wave only)
  const int32_t* lengths;            // (B,), nullable
  int64_t xt, xb, at, ab, ht, hb, dht, dhb;   // elements between steps / rows of x (and dx), alpha (and dalpha), h, dh
  int64_t dxt, dxb, dat, dab;
  int T, B, D, G, reverse;
  int tiles, chunks, tiles_per_chunk;
};

// ---- gates --------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float gate_of(float alpha) {
  const float s = fminf(fmaxf(alpha, -0.25f), 0.f);
  // exp(s) - 1 = s (1 + s/2 + ... + s^5/720): the next term is 5e-8 of the sum at s = -1/4
  float p = fmaf(s, 1.f / 720.f, 1.f / 120.f);
  p = fmaf(s, p, 1.f / 24.f);
  p = fmaf(s, p, 1.f / 6.f);
  p = fmaf(s, p, 0.5f);
  p = fmaf(s, p, 1.f);
  const float near = fminf(s * p, -1.17549435e-38f);              // (alpha = 0: negative all the same)
  const float far = __expf(alpha);                                // (NaN stays NaN)
  return (alpha > -0.25f && alpha <= 0.f) ? near : far;
}

// exp(alpha) h + x with q = gate_of(alpha)
__device__ __forceinline__ float gate_apply(float q, float h, float x) {
  const int bits = __float_as_int(q);
  const float kept = __int_as_float(__float_as_int(h) & (bits >> 31));
  const float hz = bits == 0 ? 0.f : h;
  return fmaf(q, hz, x) + kept;
}

// the gate of a step that leaves the state as it is (exact for every finite state)
static constexpr float kGateKeeps = -1.17549435e-38f;

constexpr int kScanW = 8, kScanU = 8, kScanTile = kScanW * kScanU;

// Which channels a lane owns.  V neighbouring ones of one row; where a gate is shared and its products have to be summed
// (GROUPED), the lanes of a gate are neighbours and no gate straddles two waves unless it is wider than one.
struct ScanLane {
  bool live;
  int64_t ch;                        // b D + c of the lane's first channel (0 for a lane without one)
  int64_t group;                     // GROUPED: b G + gate
  int b, c, gate, len, first, seg;   // first: the lane is the first of its gate in this wave
  int at, lanes;                     // GROUPED: the lane's place among the gate's lanes of this wave, and their number
};

template <int V, bool GROUPED>
__device__ __forceinline__ ScanLane scan_lane(const ScanArgs& a) {
  ScanLane l;
  const int lane = threadIdx.x & 63, per = a.D / a.G;
  l.group = 0; l.seg = 0; l.at = 0; l.lanes = 1; l.first = 1;
  if constexpr (GROUPED) {
    const int wide = per / V;        // lanes of a gate
    if (wide <= 64) {
      const int fit = 64 / wide;
      l.group = (int64_t)blockIdx.x * fit + lane / wide;
      l.at = lane % wide;
      l.lanes = wide;
      l.live = lane / wide < fit && l.group < (int64_t)a.B * a.G;
      l.c = l.at * V;
    } else {
      const int segs = (wide + 63) / 64;
      l.group = blockIdx.x / segs;
      l.seg = blockIdx.x % segs;
      l.at = lane;
      l.lanes = min(64, wide - l.seg * 64);
      l.live = lane < l.lanes;
      l.c = (l.seg * 64 + lane) * V;
    }
    if (!l.live) { l.group = 0; l.c = 0; }
    l.first = l.at == 0;
    l.b = (int)(l.group / a.G);
    l.gate = (int)(l.group % a.G);
    l.c += l.gate * per;
    l.ch = (int64_t)l.b * a.D + l.c;
  } else {
    l.ch = ((int64_t)blockIdx.x * 64 + lane) * V;
    l.live = l.ch < (int64_t)a.B * a.D;
    if (!l.live) l.ch = 0;
    l.b = (int)(l.ch / a.D);
    l.c = (int)(l.ch % a.D);
    l.gate = l.c / per;
  }
  l.len = a.lengths ? min(max(a.lengths[l.b], 0), a.T) : a.T;
  if (!l.live) l.len = 0;
  return l;
}

// the address of a row's step 0, and the distance from a step to the next one, in the row's direction
template <typename T>
__device__ __forceinline__ T* scan_origin(T* p, const ScanArgs& a, const ScanLane& l, int64_t st, int64_t sb, int c) {
  return p + (int64_t)l.b * sb + c + (a.reverse && l.len > 0 ? (int64_t)(l.len - 1) * st : 0);
}

// U steps from step k0 on, V values each; nothing is read behind the length
template <typename T, int V, int U>
__device__ __forceinline__ void scan_load(reg_vec<T, V> (&out)[U], const T* origin, int64_t d, int k0, int len, bool full) {
  const T* p = origin + (int64_t)k0 * d;
  if (full) {
#pragma unroll
    for (int u = 0; u < U; ++u) out[u] = load_vec<T, V>(p + u * d);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u < len) out[u] = load_vec<T, V>(p + u * d);
    }
  }
}

// q of every step of a run and the sum of its alphas (-inf once a gate forgets)
template <typename TA, int NA, int U>
__device__ __forceinline__ void scan_gates(float (&q)[U][NA], float (&sum)[NA], const reg_vec<TA, NA> (&raw)[U], int k0, int len) {
#pragma unroll
  for (int i = 0; i < NA; ++i) sum[i] = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const float alpha = raw[u][i];
      const bool in = k0 + u < len;
      q[u][i] = in ? gate_of(alpha) : kGateKeeps;
      sum[i] += !in ? 0.f : q[u][i] == 0.f ? -__builtin_inff() : alpha;
    }
}

// The state in front of chunk `chunk`, from the runs of the chunks in front of it (behind it, for the backward).
template <int V>
__device__ __forceinline__ void scan_compose(float (&s)[V], const ScanArgs& a, const ScanLane& l, int from, int to, int by) {
  const int64_t C = (int64_t)a.B * a.D;
  for (int j = from; j != to; j += by) {
    const float* p = a.run + (int64_t)j * 2 * C + l.ch;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = gate_apply(gate_of(p[i]), s[i], p[C + i]);
  }
}

// FINAL: the whole forward.  Not FINAL: (S, l) of every chunk but the last.
template <typename T, typename TA, int V, int NA, bool FINAL>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_fwd_kernel(const ScanArgs a) {
  constexpr int U = kScanU, W = kScanW;
  __shared__ float exq[2][W][NA][64], exl[2][W][V][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const ScanLane l = scan_lane<V, false>(a);
  const int64_t C = (int64_t)a.B * a.D;
  const int chunk = blockIdx.y, tile0 = chunk * a.tiles_per_chunk, tile1 = min(tile0 + a.tiles_per_chunk, a.tiles);
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, dh = a.reverse ? -a.ht : a.ht;
  const T* x0 = scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c);
  const TA* a0 = scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, NA == 1 ? l.gate : l.c);
  T* h0 = scan_origin(static_cast<T*>(a.h), a, l, a.ht, a.hb, l.c);
  T* pad = static_cast<T*>(a.h) + (int64_t)l.b * a.hb + l.c;        // steps behind the length lie at their own index

  float carry[V], total[NA];
#pragma unroll
  for (int i = 0; i < V; ++i) carry[i] = FINAL && a.initial && l.live ? a.initial[l.ch + i] : 0.f;
#pragma unroll
  for (int i = 0; i < NA; ++i) total[i] = 0.f;
  if constexpr (FINAL) scan_compose<V>(carry, a, l, 0, chunk, 1);

  reg_vec<T, V> rx[U];
  reg_vec<TA, NA> ra[U];
  auto fetch = [&](int tile) {
    const int k0 = (tile * W + wave) * U;
    const bool full = __all(k0 + U <= l.len);
    scan_load<T, V, U>(rx, x0, dx, k0, l.len, full);
    scan_load<TA, NA, U>(ra, a0, da, k0, l.len, full);
  };
  fetch(tile0);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int k0 = (tile * W + wave) * U, buf = tile & 1;
    float x[U][V], q[U][NA], sum[NA], run[V];
    scan_gates<TA, NA, U>(q, sum, ra, k0, l.len);
#pragma unroll
    for (int i = 0; i < V; ++i) run[i] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[u][i] = k0 + u < l.len ? rx[u][i] : 0.f;
        run[i] = gate_apply(q[u][NA == 1 ? 0 : i], run[i], x[u][i]);
      }
    if (tile + 1 < tile1) fetch(tile + 1);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      exq[buf][wave][i][lane] = gate_of(sum[i]);
      total[i] += sum[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) exl[buf][wave][i][lane] = run[i];
    __syncthreads();
    if (FINAL && a.state && wave == 0 && l.live) {
#pragma unroll
      for (int i = 0; i < V; ++i) a.state[(int64_t)tile * C + l.ch + i] = carry[i];
    }
    float h[V];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (w == wave) h[i] = carry[i];
        carry[i] = gate_apply(exq[buf][w][NA == 1 ? 0 : i][lane], carry[i], exl[buf][w][i][lane]);
      }
    if constexpr (FINAL) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u;
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = gate_apply(q[u][NA == 1 ? 0 : i], h[i], x[u][i]);
        if (k < l.len) {
          store_vec<T, V>(h0 + (int64_t)k * dh, h);
        } else if (l.live && k < a.T) {
          const float zero[V] = {};
          store_vec<T, V>(pad + (int64_t)k * a.ht, zero);
        }
      }
    }
  }
  if constexpr (FINAL) {
    if (a.final && chunk == a.chunks - 1 && wave == 0 && l.live) {
#pragma unroll
      for (int i = 0; i < V; ++i) a.final[l.ch + i] = carry[i];
    }
  } else {
    // the chunk's S: the waves' sums, added in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NA; ++i) exq[0][wave][i][lane] = total[i];
    __syncthreads();
    if (wave == 0 && l.live) {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        total[i] = 0.f;
        for (int w = 0; w < W; ++w) total[i] += exq[0][w][i][lane];
      }
      float* p = a.run + (int64_t)chunk * 2 * C + l.ch;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] = total[NA == 1 ? 0 : i];
        p[C + i] = carry[i];
      }
    }
  }
}

// The sum over a gate's lanes of this wave, in the lane `at` = 0.  A power of two of them lies on its own boundary.
__device__ __forceinline__ float gate_lanes_sum(float v, int at, int lanes) {
  switch (lanes) {
    case 1: return v;
    case 2: return lanes_sum<2>(v);
    case 4: return lanes_sum<4>(v);
    case 8: return lanes_sum<8>(v);
    case 16: return lanes_sum<16>(v);
    case 32: return lanes_sum<32>(v);
    case 64: return lanes_sum<64>(v);
    default: break;
  }
  int off = 1;
  while (off * 2 < lanes) off *= 2;
  for (; off > 0; off /= 2) {
    const float other = __shfl_down(v, off, 64);
    if (at + off < lanes) v += other;
  }
  return v;
}

// FINAL: the whole backward.  Not FINAL: (S, l) of every chunk but the first.
// GROUPED: a gate has several channels (NA = 1); otherwise every channel has its own (NA = V).
template <typename T, typename TA, int V, int NA, bool GROUPED, bool FINAL>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_bwd_kernel(const ScanArgs a) {
  constexpr int U = kScanU, W = kScanW;
  __shared__ float exq[2][W][NA][64], exl[2][W][V][64], exg[2][W][V][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const ScanLane l = scan_lane<V, GROUPED>(a);
  const int64_t C = (int64_t)a.B * a.D;
  const int chunk = blockIdx.y + (FINAL ? 0 : 1), tile0 = chunk * a.tiles_per_chunk, tile1 = min(tile0 + a.tiles_per_chunk, a.tiles);
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, ddh = a.reverse ? -a.dht : a.dht;
  const int64_t ddx = a.reverse ? -a.dxt : a.dxt, dda = a.reverse ? -a.dat : a.dat;
  const int gate = NA == 1 ? l.gate : l.c;
  const T* x0 = scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c);
  const T* d0 = scan_origin(static_cast<const T*>(a.dh), a, l, a.dht, a.dhb, l.c);
  const TA* a0 = scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, gate);
  T* gx0 = scan_origin(static_cast<T*>(a.dx), a, l, a.dxt, a.dxb, l.c);
  T* padx = static_cast<T*>(a.dx) + (int64_t)l.b * a.dxb + l.c;
  TA* ga0 = scan_origin(static_cast<TA*>(a.dalpha), a, l, a.dat, a.dab, gate);
  TA* pada = static_cast<TA*>(a.dalpha) + (int64_t)l.b * a.dab + gate;
  const int segs = GROUPED ? (a.D / a.G / V + 63) / 64 : 1;

  float carry[V], total[NA];
#pragma unroll
  for (int i = 0; i < V; ++i) carry[i] = FINAL && a.dfinal && l.live ? a.dfinal[l.ch + i] : 0.f;
#pragma unroll
  for (int i = 0; i < NA; ++i) total[i] = 0.f;
  if constexpr (FINAL) scan_compose<V>(carry, a, l, a.chunks - 1, chunk, -1);

  reg_vec<T, V> rx[U], rd[U];
  reg_vec<TA, NA> ra[U];
  auto fetch = [&](int tile) {
    const int k0 = (tile * W + wave) * U;
    const bool full = __all(k0 + U <= l.len);
    if constexpr (FINAL) scan_load<T, V, U>(rx, x0, dx, k0, l.len, full);
    if (a.dh) scan_load<T, V, U>(rd, d0, ddh, k0, l.len, full);
    scan_load<TA, NA, U>(ra, a0, da, k0, l.len, full);
  };
  fetch(tile1 - 1);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    const int k0 = (tile * W + wave) * U, buf = tile & 1;
    float x[U][V], d[U][V], q[U][NA], sum[NA], run[V], back[V], h[V], g[V];
    scan_gates<TA, NA, U>(q, sum, ra, k0, l.len);
#pragma unroll
    for (int i = 0; i < V; ++i) run[i] = back[i] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (FINAL) {
          x[u][i] = k0 + u < l.len ? rx[u][i] : 0.f;
          run[i] = gate_apply(q[u][NA == 1 ? 0 : i], run[i], x[u][i]);
        }
        d[u][i] = a.dh && k0 + u < l.len ? rd[u][i] : 0.f;
      }
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int i = 0; i < V; ++i) back[i] = gate_apply(q[u][NA == 1 ? 0 : i], back[i] + d[u][i], 0.f);
    if (tile > tile0) fetch(tile - 1);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = FINAL && l.live ? a.state[(int64_t)tile * C + l.ch + i] : 0.f;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      exq[buf][wave][i][lane] = gate_of(sum[i]);
      total[i] += sum[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (FINAL) exl[buf][wave][i][lane] = run[i];
      exg[buf][wave][i][lane] = back[i];
    }
    __syncthreads();
    if constexpr (FINAL) {
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (w < wave) h[i] = gate_apply(exq[buf][w][NA == 1 ? 0 : i][lane], h[i], exl[buf][w][i][lane]);
    }
#pragma unroll
    for (int w = W - 1; w >= 0; --w)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (w == wave) g[i] = carry[i];
        carry[i] = gate_apply(exq[buf][w][NA == 1 ? 0 : i][lane], carry[i], exg[buf][w][i][lane]);
      }
    if constexpr (FINAL) {
      // x becomes a_k h_{k-1}
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float p = gate_apply(q[u][NA == 1 ? 0 : i], h[i], 0.f);
          h[i] = p + x[u][i];
          x[u][i] = p;
        }
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        const int k = k0 + u;
        float gx[V], galpha[NA];
#pragma unroll
        for (int i = 0; i < NA; ++i) galpha[i] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          gx[i] = g[i] + d[u][i];
          galpha[NA == 1 ? 0 : i] += x[u][i] * gx[i];
          g[i] = gate_apply(q[u][NA == 1 ? 0 : i], gx[i], 0.f);
        }
        const bool in = k < l.len, behind = !in && l.live && k < a.T;
        if (in) {
          store_vec<T, V>(gx0 + (int64_t)k * ddx, gx);
        } else if (behind) {
          const float zero[V] = {};
          store_vec<T, V>(padx + (int64_t)k * a.dxt, zero);
        }
        if constexpr (GROUPED) {
          const float s = gate_lanes_sum(in ? galpha[0] : 0.f, l.at, l.lanes);
          const float out[1] = {s};
          if (l.first && segs > 1) {
            const int64_t t = in && a.reverse ? l.len - 1 - k : k;
            if (in || behind) a.part[(t * a.B * a.G + l.group) * segs + l.seg] = s;
          } else if (l.first && in) {
            store_vec<TA, 1>(ga0 + (int64_t)k * dda, out);
          } else if (l.first && behind) {
            store_vec<TA, 1>(pada + (int64_t)k * a.dat, out);
          }
        } else if (in) {
          store_vec<TA, NA>(ga0 + (int64_t)k * dda, galpha);
        } else if (behind) {
          const float zero[NA] = {};
          store_vec<TA, NA>(pada + (int64_t)k * a.dat, zero);
        }
      }
    }
  }
  if constexpr (FINAL) {
    if (a.dinitial && chunk == 0 && wave == 0 && l.live) {
#pragma unroll
      for (int i = 0; i < V; ++i) a.dinitial[l.ch + i] = carry[i];
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NA; ++i) exq[0][wave][i][lane] = total[i];
    __syncthreads();
    if (wave == 0 && l.live) {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        total[i] = 0.f;
        for (int w = 0; w < W; ++w) total[i] += exq[0][w][i][lane];
      }
      float* p = a.run + (int64_t)chunk * 2 * C + l.ch;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] = total[NA == 1 ? 0 : i];
        p[C + i] = carry[i];
      }
    }
  }
}

// adds the waves' partial sums of gates wider than a wave
template <typename TA>
__global__ __launch_bounds__(256) void gated_scan_bwd_finish_kernel(const ScanArgs a, int segs) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, groups = (int64_t)a.B * a.G;
  if (i >= a.T * groups) return;
  float s = 0.f;
  for (int k = 0; k < segs; ++k) s += a.part[i * segs + k];
  const int64_t t = i / groups, group = i % groups;
  static_cast<TA*>(a.dalpha)[t * a.dat + group / a.G * a.dab + group % a.G] = (TA)s;
}

// one step on a state that stays: state = exp(alpha) state + x, h = state
template <typename T, typename TA>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(const T* __restrict__ x, const TA* __restrict__ alpha, float* __restrict__ state,
                                                              T* __restrict__ h, int B, int D, int per, int64_t xb, int64_t ab, int64_t sb) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)B * D) return;
  const int64_t b = i / D;
  const int c = (int)(i - b * D);
  float* s = state + b * sb + c;
  const float v = gate_apply(gate_of((float)alpha[b * ab + c / per]), *s, (float)x[b * xb + c]);
  *s = v;
  h[i] = (T)v;
}

// ---- launches ------------------------------------------------------------------------------------------------------------------
struct ScanPlan {
  int V, tiles, chunks, tiles_per_chunk, segs;
  int64_t fwd_blocks, bwd_blocks;
};

// V = 4 or 2 channels a lane where they divide the channels of a row (of a gate) and the chip stays busy; time in chunks where
// the channels alone make fewer than 512 workgroups, two for every CU, and a chunk keeps four tiles or more.
static ScanPlan scan_plan(const socmx_scan& s) {
  ScanPlan p;
  const int64_t C = (int64_t)s.B * s.D;
  const int per = s.D / s.G;
  p.V = 1;
  for (int v = 4; v > 1; v /= 2)
    if (s.D % v == 0 && (per == 1 || per % v == 0) && C / (64 * v) >= 64) { p.V = v; break; }
  p.fwd_blocks = (C + 64 * p.V - 1) / (64 * p.V);
  p.segs = 1;
  p.bwd_blocks = p.fwd_blocks;
  if (per > 1) {
    const int wide = per / p.V;
    p.segs = wide <= 64 ? 1 : (wide + 63) / 64;
    const int64_t groups = (int64_t)s.B * s.G;
    p.bwd_blocks = wide <= 64 ? (groups + 64 / wide - 1) / (64 / wide) : groups * p.segs;
  }
  p.tiles = (s.T + kScanTile - 1) / kScanTile;
  const int64_t want = (512 + p.fwd_blocks - 1) / p.fwd_blocks;
  p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>({want, p.tiles / 4, 64}));
  p.tiles_per_chunk = (p.tiles + p.chunks - 1) / p.chunks;
  p.chunks = (p.tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk;
  return p;
}

static int scan_check(const socmx_scan* s) {
  if (!s) return SOCMX_E_NULL;
  if (s->type < SOCMX_F32 || s->type > SOCMX_F16 || (s->gate_type != s->type && s->gate_type != SOCMX_F32)) return SOCMX_E_KIND;
  if (s->T < 1 || s->B < 1 || s->D < 1 || s->G < 1 || s->D % s->G != 0) return SOCMX_E_DIM;
  if (s->T > (1 << 30) || (int64_t)s->B * s->D > (1ll << 31)) return SOCMX_E_DIM;
  return 0;
}

static ScanArgs scan_args(const socmx_scan& s, const ScanPlan& p) {
  ScanArgs a = {};
  a.lengths = s.lengths;
  a.xt = s.x_stride_t; a.xb = s.x_stride_b; a.at = s.gate_stride_t; a.ab = s.gate_stride_b;
  a.T = s.T; a.B = s.B; a.D = s.D; a.G = s.G; a.reverse = s.reverse != 0;
  a.tiles = p.tiles; a.chunks = p.chunks; a.tiles_per_chunk = p.tiles_per_chunk;
  return a;
}

template <typename T, typename TA, int V, bool BWD>
static int launch_scan(const ScanArgs& a, const ScanPlan& p, void* stream) {
  const bool own = a.G == a.D;
  const dim3 block(64 * kScanW);
  const unsigned n = (unsigned)(BWD ? p.bwd_blocks : p.fwd_blocks);
  int err = 0;
  if constexpr (!BWD) {
    if (p.chunks > 1)
      err = own ? launch(gated_scan_fwd_kernel<T, TA, V, V, false>, dim3(n, p.chunks - 1), block, 0, stream, a)
                : launch(gated_scan_fwd_kernel<T, TA, V, 1, false>, dim3(n, p.chunks - 1), block, 0, stream, a);
    if (err) return err;
    return own ? launch(gated_scan_fwd_kernel<T, TA, V, V, true>, dim3(n, p.chunks), block, 0, stream, a)
               : launch(gated_scan_fwd_kernel<T, TA, V, 1, true>, dim3(n, p.chunks), block, 0, stream, a);
  } else {
    if (p.chunks > 1)
      err = own ? launch(gated_scan_bwd_kernel<T, TA, V, V, false, false>, dim3(n, p.chunks - 1), block, 0, stream, a)
                : launch(gated_scan_bwd_kernel<T, TA, V, 1, true, false>, dim3(n, p.chunks - 1), block, 0, stream, a);
    if (err) return err;
    err = own ? launch(gated_scan_bwd_kernel<T, TA, V, V, false, true>, dim3(n, p.chunks), block, 0, stream, a)
              : launch(gated_scan_bwd_kernel<T, TA, V, 1, true, true>, dim3(n, p.chunks), block, 0, stream, a);
    if (err || p.segs == 1) return err;
    const int64_t sums = (int64_t)a.T * a.B * a.G;
    return launch(gated_scan_bwd_finish_kernel<TA>, dim3((unsigned)((sums + 255) / 256)), dim3(256), 0, stream, a, p.segs);
  }
}

template <typename T, typename TA, bool BWD>
static int launch_scan_v(const ScanArgs& a, const ScanPlan& p, void* stream) {
  if (p.V == 4) return launch_scan<T, TA, 4, BWD>(a, p, stream);
  if (p.V == 2) return launch_scan<T, TA, 2, BWD>(a, p, stream);
  return launch_scan<T, TA, 1, BWD>(a, p, stream);
}

template <bool BWD>
static int dispatch_scan(const socmx_scan& s, const ScanArgs& a, const ScanPlan& p, void* stream) {
  const bool wide = s.gate_type == SOCMX_F32;
  if (s.type == SOCMX_F32) return launch_scan_v<float, float, BWD>(a, p, stream);
  if (s.type == SOCMX_BF16) return wide ? launch_scan_v<bf16_t, float, BWD>(a, p, stream) : launch_scan_v<bf16_t, bf16_t, BWD>(a, p, stream);
  return wide ? launch_scan_v<f16_t, float, BWD>(a, p, stream) : launch_scan_v<f16_t, f16_t, BWD>(a, p, stream);
}

}  // namespace socmx

using namespace socmx;

extern "C" int socmx_gated_scan_sizes(const socmx_scan* scan, int64_t* state_floats, int64_t* fwd_workspace_floats,
                                      int64_t* bwd_workspace_floats) {
  if (const int bad = scan_check(scan)) return bad;
  if (!state_floats || !fwd_workspace_floats || !bwd_workspace_floats) return SOCMX_E_NULL;
  const ScanPlan p = scan_plan(*scan);
  const int64_t C = (int64_t)scan->B * scan->D, runs = p.chunks > 1 ? p.chunks * 2 * C : 0;
  *state_floats = p.tiles * C;
  *fwd_workspace_floats = runs;
  *bwd_workspace_floats = runs + (p.segs > 1 ? (int64_t)scan->T * scan->B * scan->G * p.segs : 0);
  return 0;
}

extern "C" int socmx_gated_scan_fwd(const socmx_scan* scan, const void* x, const void* log_decay, const float* initial, void* h,
                                    int64_t h_stride_t, int64_t h_stride_b, float* final_state, float* states, float* workspace,
                                    socmx_stream_t stream) {
  if (const int bad = scan_check(scan)) return bad;
  if (!x || !log_decay || !h) return SOCMX_E_NULL;
  const ScanPlan p = scan_plan(*scan);
  if (p.chunks > 1 && !workspace) return SOCMX_E_WORKSPACE;
  ScanArgs a = scan_args(*scan, p);
  a.x = x; a.alpha = log_decay; a.initial = initial; a.h = h; a.ht = h_stride_t; a.hb = h_stride_b;
  a.final = final_state; a.state = states; a.run = workspace;
  return dispatch_scan<false>(*scan, a, p, stream);
}

extern "C" int socmx_gated_scan_bwd(const socmx_scan* scan, const void* x, const void* log_decay, const float* states, const void* dh,
                                    int64_t dh_stride_t, int64_t dh_stride_b, const float* dfinal, void* dx, int64_t dx_stride_t,
                                    int64_t dx_stride_b, void* dlog_decay, int64_t dgate_stride_t, int64_t dgate_stride_b,
                                    float* dinitial, float* workspace, socmx_stream_t stream) {
  if (const int bad = scan_check(scan)) return bad;
  if (!x || !log_decay || !states || !dx || !dlog_decay) return SOCMX_E_NULL;
  const ScanPlan p = scan_plan(*scan);
  if ((p.chunks > 1 || p.segs > 1) && !workspace) return SOCMX_E_WORKSPACE;
  ScanArgs a = scan_args(*scan, p);
  a.x = x; a.alpha = log_decay; a.state = const_cast<float*>(states); a.dh = dh; a.dht = dh_stride_t; a.dhb = dh_stride_b;
  a.dfinal = dfinal; a.dx = dx; a.dxt = dx_stride_t; a.dxb = dx_stride_b;
  a.dalpha = dlog_decay; a.dat = dgate_stride_t; a.dab = dgate_stride_b; a.dinitial = dinitial;
  a.run = workspace;
  a.part = workspace ? workspace + (p.chunks > 1 ? (int64_t)p.chunks * 2 * scan->B * scan->D : 0) : nullptr;
  return dispatch_scan<true>(*scan, a, p, stream);
}

extern "C" int socmx_gated_scan_step(int32_t type, int32_t gate_type, int32_t B, int32_t D, int32_t G, const void* x, int64_t x_stride,
                                     const void* log_decay, int64_t gate_stride, float* state, int64_t state_stride, void* h,
                                     socmx_stream_t stream) {
  if (!x || !log_decay || !state || !h) return SOCMX_E_NULL;
  if (type < SOCMX_F32 || type > SOCMX_F16 || (gate_type != type && gate_type != SOCMX_F32)) return SOCMX_E_KIND;
  if (B < 1 || D < 1 || G < 1 || D % G != 0 || (int64_t)B * D > (1ll << 31)) return SOCMX_E_DIM;
  const dim3 grid((unsigned)(((int64_t)B * D + 255) / 256)), block(256);
  const int per = D / G;
#define SOCMX_STEP(T, TA) \
  launch(gated_scan_step_kernel<T, TA>, grid, block, 0, stream, (const T*)x, (const TA*)log_decay, state, (T*)h, B, D, per, x_stride, \
         gate_stride, state_stride)
  if (type == SOCMX_F32) return SOCMX_STEP(float, float);
  if (type == SOCMX_BF16) return gate_type == SOCMX_F32 ? SOCMX_STEP(bf16_t, float) : SOCMX_STEP(bf16_t, bf16_t);
  return gate_type == SOCMX_F32 ? SOCMX_STEP(f16_t, float) : SOCMX_STEP(f16_t, f16_t);
#undef SOCMX_STEP
}
