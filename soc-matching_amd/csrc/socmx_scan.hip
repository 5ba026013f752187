// socmx_scan.hip -- the gated linear recurrence along a trajectory, forward, backward and one step, gfx950.
//
//   h_t = a_t h_{t-1} + x_t,   a_t = exp(alpha_t),   h_{-1} = initial          x, h (T, B, D);  alpha (T, B, G), a gate per D / G channels
//   G_t = dh_t + a_{t+1} G_{t+1}:   dx_t = G_t,   dalpha_t = a_t h_{t-1} G_t (summed over a gate's channels),   dinitial = a_0 G_0
// in either direction of time (`reverse`) and up to a length of its own for every row b (`lengths`): "step k" below is the row's
// k-th step in its direction, the steps behind its length leave the state alone and get zeros.
//
// THE GATE.  A memory of n steps has a = 1 - 1/n: rounding a to f32 moves the steady state x / (1 - a) by n 2^-25, the same way
// on every step of a constant decay.  So a gate near 1 (-1/4 < alpha <= 0) is kept as q = exp(alpha) - 1 (a polynomial, full relative
// precision) and r = 1, any other as q = exp(alpha) and r = 0: a h + x is q h + x, plus r h, two fused operations.  q = 0 (exp flushes
// what is below 2^-126) is a gate that forgets: whatever stood before it, infinities and NaN included, is replaced, not multiplied.
//
// RUNS.  A step is an affine map, so a run of steps is one: h -> exp(S) h + l with S the sum of its alphas and l its result from zero --
// the same form, applied with the code of a step.  A wave owns 64 V channels and a run of steps, and walks it alone, U steps at a time
// with the next U in flight: no barrier, nothing but the state between two steps.  Where the channels do not fill the chip, time is
// cut into runs: a first launch forms every run's (S, l), W of them a workgroup, and the composition of those W; the second composes the
// workgroups in front of its own, then the waves, and walks its run from the state it found.  x and alpha are read twice for that,
// the second time mostly out of the last-level cache: the second launch takes the runs in the opposite order.  (A form whose
// waves met in LDS every 64 steps took 329 us against 215 at (4096, 8, 2048) bf16 with 32 gates and padded rows, forward and backward, and
// 450 against 435 at (65536, 1, 640) f32.)
//
// THE BACKWARD walks the steps from the end.  It rebuilds U steps of h at a time in f32 from the states that the forward leaves every
// U steps (f32, 1 / U of h) -- h itself, rounded to 16 bits, would put its rounding into dalpha.  A gate shared by several channels: their
// products are summed across the lanes in a fixed order, gates wider than a wave leave one partial sum a wave for another launch.  No
// atomics: the same bits on every run.  Bound by memory: x, alpha (, dh) in, h (dx, dalpha) out.
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
  float* state;                      // (ceil(T / U), B D): the state in front of every U-th step; written by the forward when not NULL
  float* run;                        // (chunks, 1 + W, 2, B D): q and l of a workgroup's steps, then of each of its waves' (chunked only)
  float* part;                       // (T, B G, segments): partial sums of dalpha (gates wider than a wave only)
  const int32_t* lengths;            // (B,), nullable
  int64_t xt, xb, at, ab, ht, hb, dht, dhb;   // elements between steps / rows of x, alpha, h, dh
  int64_t dxt, dxb, dat, dab;                 // of dx, dalpha
  int T, B, D, G, reverse;
  int steps, chunks;                 // steps of a run (a multiple of U), workgroups of W runs along time
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
__device__ __forceinline__ float gate_keeps(float q) { return q < 0.f ? 1.f : 0.f; }

// the gate of a step that leaves the state as it is (exact for every finite state)
static constexpr float kGateKeeps = -1.17549435e-38f;

// a h + x.  CUT: the gate may forget
template <bool CUT>
__device__ __forceinline__ float gate_apply(float q, float r, float h, float x) {
  if (CUT) h = q == 0.f ? 0.f : h;
  return fmaf(r, h, fmaf(q, h, x));
}
template <bool CUT>
__device__ __forceinline__ float gate_times(float q, float r, float h) {
  if (CUT) h = q == 0.f ? 0.f : h;
  return fmaf(r, h, q * h);
}
__device__ __forceinline__ float gate_apply(float q, float h, float x) { return gate_apply<true>(q, gate_keeps(q), h, x); }

constexpr int kScanW = 8, kScanU = 8;

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
  if (!l.live) l.len = a.T;            // (a lane without channels walks along with channel 0 and stores nothing)
  return l;
}

// where a wave's steps end: at `end`, or at the first multiple of U behind the last step that one of its rows has
__device__ __forceinline__ int scan_stop(const ScanLane& l, int begin, int end) {
  int most = l.live ? l.len : 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off, 64));
  return max(begin, min(end, (most + kScanU - 1) / kScanU * kScanU));
}

// zeros at the steps [from, to) of a lane's V channels (or its gates), which lie behind the lengths
template <typename T, int V>
__device__ __forceinline__ void scan_clear(T* origin, int64_t st, int from, int to) {
  const float zero[V] = {};
  for (int k = from; k < to; ++k) store_vec<T, V>(origin + (int64_t)k * st, zero);
}

// the address of a row's step 0, and the distance from a step to the next one, in the row's direction
template <typename T>
__device__ __forceinline__ T* scan_origin(T* p, const ScanArgs& a, const ScanLane& l, int64_t st, int64_t sb, int c) {
  return p + (int64_t)l.b * sb + c + (a.reverse && l.len > 0 ? (int64_t)(l.len - 1) * st : 0);
}

// U steps from step k0 on, V values each; nothing is read behind the length
template <typename T, int V>
__device__ __forceinline__ void scan_load(reg_vec<T, V> (&out)[kScanU], const T* origin, int64_t d, int k0, int len, bool full) {
  const T* p = origin + (int64_t)k0 * d;
  if (full) {
#pragma unroll
    for (int u = 0; u < kScanU; ++u) out[u] = load_vec<T, V>(p + u * d);
  } else {
#pragma unroll
    for (int u = 0; u < kScanU; ++u)
      if (k0 + u < len) out[u] = load_vec<T, V>(p + u * d);
  }
}

template <typename T, int V>
__device__ __forceinline__ void scan_values(float (&out)[kScanU][V], const reg_vec<T, V> (&raw)[kScanU], int k0, int len, bool full) {
  if (full) {
#pragma unroll
    for (int u = 0; u < kScanU; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) out[u][i] = raw[u][i];
  } else {
#pragma unroll
    for (int u = 0; u < kScanU; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) out[u][i] = k0 + u < len ? raw[u][i] : 0.f;
  }
}

// q and r of U steps; whether one of this wave's gates forgets
template <typename TA, int NA>
__device__ __forceinline__ bool scan_gates(float (&q)[kScanU][NA], float (&r)[kScanU][NA], const reg_vec<TA, NA> (&raw)[kScanU], int k0, int len,
                                           bool full) {
  bool cut = false;
#pragma unroll
  for (int u = 0; u < kScanU; ++u)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      q[u][i] = gate_of(raw[u][i]);
      if (!full && k0 + u >= len) q[u][i] = kGateKeeps;
      r[u][i] = gate_keeps(q[u][i]);
      cut |= q[u][i] == 0.f;
    }
  return __any(cut);
}

// the sum of a run's alphas, -inf once a gate forgets
template <typename TA, int NA>
__device__ __forceinline__ void scan_sum(float (&sum)[NA], const float (&q)[kScanU][NA], const reg_vec<TA, NA> (&raw)[kScanU], int k0, int len,
                                         bool full) {
#pragma unroll
  for (int u = 0; u < kScanU; ++u)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const float alpha = !full && k0 + u >= len ? 0.f : (float)raw[u][i];
      sum[i] += q[u][i] == 0.f ? -__builtin_inff() : alpha;
    }
}

// the state in front of (behind, for the backward) a wave's run, from the runs of the workgroups and then the waves before it
template <int V>
__device__ __forceinline__ void scan_compose(float (&s)[V], const ScanArgs& a, int64_t ch, int chunk, int wave, int first_chunk, int first_wave) {
  const int64_t C = (int64_t)a.B * a.D, row = 2 * C, step = (1 + kScanW) * row;
  const int by = first_chunk <= chunk ? 1 : -1;
#pragma unroll 4
  for (int j = first_chunk; j != chunk; j += by) {
    const float* p = a.run + j * step + ch;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = gate_apply(p[i], s[i], p[C + i]);
  }
  const int wby = first_wave <= wave ? 1 : -1;
  for (int w = first_wave; w != wave; w += wby) {
    const float* p = a.run + chunk * step + (1 + w) * row + ch;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = gate_apply(p[i], s[i], p[C + i]);
  }
}

// a wave's run (S, l) to memory, and the composition of its workgroup's: in the order of the steps, or against it (back)
template <int V, int NA>
__device__ __forceinline__ void scan_runs(const ScanArgs& a, const ScanLane& l, int chunk, const float (&sum)[NA], const float (&run)[V], bool back) {
  __shared__ float exs[kScanW][NA][64], exl[kScanW][V][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t C = (int64_t)a.B * a.D;
  float* p = a.run + (int64_t)chunk * (1 + kScanW) * 2 * C + l.ch;
#pragma unroll
  for (int i = 0; i < NA; ++i) exs[wave][i][lane] = sum[i];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    exl[wave][i][lane] = run[i];
    if (l.live) {
      p[(1 + wave) * 2 * C + i] = gate_of(sum[NA == 1 ? 0 : i]);
      p[(1 + wave) * 2 * C + C + i] = run[i];
    }
  }
  __syncthreads();
  if (wave == 0 && l.live) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = 0.f, all = 0.f;
#pragma unroll
      for (int k = 0; k < kScanW; ++k) {
        const int w = back ? kScanW - 1 - k : k;
        const float one = exs[w][NA == 1 ? 0 : i][lane];
        s = gate_apply(gate_of(one), s, exl[w][i][lane]);
        all += one;
      }
      p[i] = gate_of(all);
      p[C + i] = s;
    }
  }
}

// the first launch of a forward in chunks: the runs of all of them but the last
template <typename T, typename TA, int V, int NA>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_fwd_runs_kernel(const ScanArgs a) {
  const int wave = threadIdx.x >> 6, chunk = blockIdx.y;
  const ScanLane l = scan_lane<V, false>(a);
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at;
  const T* x0 = scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c);
  const TA* a0 = scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, NA == 1 ? l.gate : l.c);
  const int begin = (chunk * kScanW + wave) * a.steps, end = min(begin + a.steps, a.T);
  float sum[NA] = {}, run[V] = {};
  reg_vec<T, V> rx[kScanU];
  reg_vec<TA, NA> ra[kScanU];
  auto fetch = [&](int k0) {
    const bool full = __all(k0 + kScanU <= l.len);
    scan_load<T, V>(rx, x0, dx, k0, l.len, full);
    scan_load<TA, NA>(ra, a0, da, k0, l.len, full);
  };
  const int stop = scan_stop(l, begin, end);
  if (begin < stop) fetch(begin);
  for (int k0 = begin; k0 < stop; k0 += kScanU) {
    const bool full = __all(k0 + kScanU <= l.len);
    float x[kScanU][V], q[kScanU][NA], r[kScanU][NA];
    scan_values<T, V>(x, rx, k0, l.len, full);
    const bool cut = scan_gates<TA, NA>(q, r, ra, k0, l.len, full);
    scan_sum<TA, NA>(sum, q, ra, k0, l.len, full);
    if (k0 + kScanU < stop) fetch(k0 + kScanU);
    auto walk = [&](auto CUT) {
#pragma unroll
      for (int u = 0; u < kScanU; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) run[i] = gate_apply<decltype(CUT)::value>(q[u][NA == 1 ? 0 : i], r[u][NA == 1 ? 0 : i], run[i], x[u][i]);
    };
    if (cut) walk(std::true_type{}); else walk(std::false_type{});
  }
  scan_runs<V, NA>(a, l, chunk, sum, run, false);
}

template <typename T, typename TA, int V, int NA>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_fwd_kernel(const ScanArgs a) {
  const int wave = threadIdx.x >> 6, chunk = a.chunks - 1 - blockIdx.y;
  const ScanLane l = scan_lane<V, false>(a);
  const int64_t C = (int64_t)a.B * a.D;
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, dh = a.reverse ? -a.ht : a.ht;
  const T* x0 = scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c);
  const TA* a0 = scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, NA == 1 ? l.gate : l.c);
  T* h0 = scan_origin(static_cast<T*>(a.h), a, l, a.ht, a.hb, l.c);
  T* pad = static_cast<T*>(a.h) + (int64_t)l.b * a.hb + l.c;        // steps behind the length lie at their own index
  const int begin = (chunk * kScanW + wave) * a.steps, end = min(begin + a.steps, a.T);
  if (begin >= end) return;
  reg_vec<T, V> rx[kScanU];
  reg_vec<TA, NA> ra[kScanU];
  auto fetch = [&](int k0) {
    const bool full = __all(k0 + kScanU <= l.len);
    scan_load<T, V>(rx, x0, dx, k0, l.len, full);
    scan_load<TA, NA>(ra, a0, da, k0, l.len, full);
  };
  const int stop = scan_stop(l, begin, end);
  if (begin < stop) fetch(begin);
  float h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = a.initial && l.live ? a.initial[l.ch + i] : 0.f;
  if (begin > 0) scan_compose<V>(h, a, l.ch, chunk, wave, 0, 0);
  for (int k0 = begin; k0 < stop; k0 += kScanU) {
    const bool full = __all(k0 + kScanU <= l.len);
    float x[kScanU][V], q[kScanU][NA], r[kScanU][NA];
    scan_values<T, V>(x, rx, k0, l.len, full);
    const bool cut = scan_gates<TA, NA>(q, r, ra, k0, l.len, full);
    if (k0 + kScanU < stop) fetch(k0 + kScanU);
    if (a.state && l.live) store_vec<float, V>(a.state + (int64_t)(k0 / kScanU) * C + l.ch, h);
    auto walk = [&](auto CUT, auto FULL) {
#pragma unroll
      for (int u = 0; u < kScanU; ++u) {
        const int k = k0 + u;
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = gate_apply<decltype(CUT)::value>(q[u][NA == 1 ? 0 : i], r[u][NA == 1 ? 0 : i], h[i], x[u][i]);
        const bool in = l.live && (decltype(FULL)::value || k < l.len);
        if (in) {
          store_vec<T, V>(h0 + (int64_t)k * dh, h);
        } else if (!decltype(FULL)::value && l.live && k < a.T) {
          const float zero[V] = {};
          store_vec<T, V>(pad + (int64_t)k * a.ht, zero);
        }
      }
    };
    if (full && !cut) walk(std::false_type{}, std::true_type{}); else walk(std::true_type{}, std::false_type{});
  }
  if (l.live) scan_clear<T, V>(pad, a.ht, stop, end);
  if (a.final && end == a.T && l.live) store_vec<float, V>(a.final + l.ch, h);
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

// the first launch of a backward in chunks: the runs of all of them but the first.  l = what comes out in front of the run for nothing
// coming in behind it
template <typename T, typename TA, int V, int NA>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_bwd_runs_kernel(const ScanArgs a) {
  const int wave = threadIdx.x >> 6, chunk = a.chunks - 1 - blockIdx.y;
  const ScanLane l = scan_lane<V, false>(a);
  const int64_t dd = a.reverse ? -a.dht : a.dht, da = a.reverse ? -a.at : a.at;
  const T* d0 = scan_origin(static_cast<const T*>(a.dh), a, l, a.dht, a.dhb, l.c);
  const TA* a0 = scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, NA == 1 ? l.gate : l.c);
  const int begin = (chunk * kScanW + wave) * a.steps, end = min(begin + a.steps, a.T);
  float sum[NA] = {}, run[V] = {};
  reg_vec<T, V> rd[kScanU];
  reg_vec<TA, NA> ra[kScanU];
  auto fetch = [&](int k0) {
    const bool full = __all(k0 + kScanU <= l.len);
    if (a.dh) scan_load<T, V>(rd, d0, dd, k0, l.len, full);
    scan_load<TA, NA>(ra, a0, da, k0, l.len, full);
  };
  const int stop = scan_stop(l, begin, end), last = stop > begin ? begin + (stop - begin - 1) / kScanU * kScanU : begin - kScanU;
  if (last >= begin) fetch(last);
  for (int k0 = last; k0 >= begin; k0 -= kScanU) {
    const bool full = __all(k0 + kScanU <= l.len);
    float d[kScanU][V], q[kScanU][NA], r[kScanU][NA];
    scan_values<T, V>(d, rd, k0, a.dh ? l.len : 0, full && a.dh);
    const bool cut = scan_gates<TA, NA>(q, r, ra, k0, l.len, full);
    scan_sum<TA, NA>(sum, q, ra, k0, l.len, full);
    if (k0 > begin) fetch(k0 - kScanU);
    auto walk = [&](auto CUT) {
#pragma unroll
      for (int u = kScanU - 1; u >= 0; --u)
#pragma unroll
        for (int i = 0; i < V; ++i) run[i] = gate_times<decltype(CUT)::value>(q[u][NA == 1 ? 0 : i], r[u][NA == 1 ? 0 : i], run[i] + d[u][i]);
    };
    if (cut) walk(std::true_type{}); else walk(std::false_type{});
  }
  scan_runs<V, NA>(a, l, chunk, sum, run, true);
}

// GROUPED: a gate has several channels (NA = 1); otherwise every channel has its own (NA = V).
template <typename T, typename TA, int V, int NA, bool GROUPED>
__global__ __launch_bounds__(64 * kScanW) void gated_scan_bwd_kernel(const ScanArgs a) {
  const int wave = threadIdx.x >> 6, chunk = blockIdx.y;
  const ScanLane l = scan_lane<V, GROUPED>(a);
  const int64_t C = (int64_t)a.B * a.D;
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, dd = a.reverse ? -a.dht : a.dht;
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
  const int begin = (chunk * kScanW + wave) * a.steps, end = min(begin + a.steps, a.T);
  if (begin >= end) return;
  const int stop = scan_stop(l, begin, end), last = stop > begin ? begin + (stop - begin - 1) / kScanU * kScanU : begin - kScanU;
  reg_vec<T, V> rx[kScanU], rd[kScanU];
  reg_vec<TA, NA> ra[kScanU];
  reg_vec<float, V> rs;
  auto fetch = [&](int k0) {
    const bool full = __all(k0 + kScanU <= l.len);
    scan_load<T, V>(rx, x0, dx, k0, l.len, full);
    if (a.dh) scan_load<T, V>(rd, d0, dd, k0, l.len, full);
    scan_load<TA, NA>(ra, a0, da, k0, l.len, full);
    rs = load_vec<float, V>(a.state + (int64_t)(k0 / kScanU) * C + l.ch);
  };
  if (last >= begin) fetch(last);
  float g[V];
#pragma unroll
  for (int i = 0; i < V; ++i) g[i] = a.dfinal && l.live ? a.dfinal[l.ch + i] : 0.f;
  if (end < a.T) scan_compose<V>(g, a, l.ch, chunk, wave, a.chunks - 1, kScanW - 1);
  for (int k0 = last; k0 >= begin; k0 -= kScanU) {
    const bool full = __all(k0 + kScanU <= l.len);
    float x[kScanU][V], d[kScanU][V], q[kScanU][NA], r[kScanU][NA], h[V];
    scan_values<T, V>(x, rx, k0, l.len, full);
    scan_values<T, V>(d, rd, k0, a.dh ? l.len : 0, full && a.dh);
    const bool cut = scan_gates<TA, NA>(q, r, ra, k0, l.len, full);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = rs[i];
    if (k0 > begin) fetch(k0 - kScanU);
    auto walk = [&](auto CUT, auto FULL) {
      constexpr bool cuts = decltype(CUT)::value, all = decltype(FULL)::value;
      // x becomes a_k h_{k-1}
#pragma unroll
      for (int u = 0; u < kScanU; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float p = gate_times<cuts>(q[u][NA == 1 ? 0 : i], r[u][NA == 1 ? 0 : i], h[i]);
          h[i] = p + x[u][i];
          x[u][i] = p;
        }
#pragma unroll
      for (int u = kScanU - 1; u >= 0; --u) {
        const int k = k0 + u;
        float gx[V], galpha[NA] = {};
#pragma unroll
        for (int i = 0; i < V; ++i) {
          gx[i] = g[i] + d[u][i];
          galpha[NA == 1 ? 0 : i] += x[u][i] * gx[i];
          g[i] = gate_times<cuts>(q[u][NA == 1 ? 0 : i], r[u][NA == 1 ? 0 : i], gx[i]);
        }
        const bool in = l.live && (all || k < l.len), behind = !all && l.live && !in && k < a.T;
        if (in) {
          store_vec<T, V>(gx0 + (int64_t)k * ddx, gx);
        } else if (behind) {
          const float zero[V] = {};
          store_vec<T, V>(padx + (int64_t)k * a.dxt, zero);
        }
        if constexpr (GROUPED) {
          const float out[1] = {gate_lanes_sum(in ? galpha[0] : 0.f, l.at, l.lanes)};
          if (l.first && segs > 1) {
            const int64_t t = in && a.reverse ? l.len - 1 - k : k;
            if (in || behind) a.part[(t * a.B * a.G + l.group) * segs + l.seg] = out[0];
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
    };
    if (full && !cut) walk(std::false_type{}, std::true_type{}); else walk(std::true_type{}, std::false_type{});
  }
  if (l.live && stop < end) {
    scan_clear<T, V>(padx, a.dxt, stop, end);
    if constexpr (!GROUPED) {
      scan_clear<TA, NA>(pada, a.dat, stop, end);
    } else if (l.first) {
      if (segs > 1)
        scan_clear<float, 1>(a.part + l.group * segs + l.seg, (int64_t)a.B * a.G * segs, stop, end);
      else
        scan_clear<TA, 1>(pada, a.dat, stop, end);
    }
  }
  if (a.dinitial && begin == 0 && l.live) store_vec<float, V>(a.dinitial + l.ch, g);
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
  int V, steps, chunks, segs;
  int64_t fwd_blocks, bwd_blocks;
};

// V channels a lane: up to 8 bytes of x and of gates of their own a step, where they divide the channels of a row (of a gate).  Runs: as
// many as give 2048 waves, two for every SIMD -- at (4096, 8, 2048) bf16 forward and backward took 375 us with 1024 waves, 285 with 1536,
// 238 with 2048, 297 with 3072, 254 with 4096: an uneven number leaves a tail, more of them read more runs -- of U steps at least, and 64
// workgroups of them along time at most, since every wave composes those in front of its own.
static ScanPlan scan_plan(const socmx_scan& s) {
  ScanPlan p;
  const int64_t C = (int64_t)s.B * s.D;
  const int per = s.D / s.G;
  p.V = 1;
  const int bytes = (s.type == SOCMX_F32 ? 4 : 2) + (per > 1 ? 0 : s.gate_type == SOCMX_F32 ? 4 : 2);
  for (int v = 4; v > 1; v /= 2)
    if (bytes * v <= 8 && s.D % v == 0 && (per == 1 || per % v == 0)) { p.V = v; break; }
  const int64_t groups = (C + 64 * p.V - 1) / (64 * p.V);
  p.fwd_blocks = p.bwd_blocks = groups;
  p.segs = 1;
  if (per > 1) {
    const int wide = per / p.V;
    p.segs = wide <= 64 ? 1 : (wide + 63) / 64;
    const int64_t gates = (int64_t)s.B * s.G;
    p.bwd_blocks = wide <= 64 ? (gates + 64 / wide - 1) / (64 / wide) : gates * p.segs;
  }
  const int64_t runs = std::max<int64_t>(1, std::min<int64_t>(2048 / groups, 64 * kScanW));
  const int64_t steps = std::max<int64_t>(kScanU, ((s.T + runs - 1) / runs + kScanU - 1) / kScanU * kScanU);
  p.steps = (int)steps;
  p.chunks = (int)((s.T + steps * kScanW - 1) / (steps * kScanW));
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
  a.steps = p.steps; a.chunks = p.chunks;
  return a;
}

// (runs are needed wherever a wave begins behind step 0, also inside the one workgroup of a short scan)
static inline bool scan_has_runs(const ScanPlan& p, int T) { return p.steps < T; }

template <typename T, typename TA, int V, bool BWD>
static int launch_scan(const ScanArgs& a, const ScanPlan& p, void* stream) {
  const bool own = a.G == a.D;
  const dim3 block(64 * kScanW), runs((unsigned)p.fwd_blocks, p.chunks), grid((unsigned)(BWD ? p.bwd_blocks : p.fwd_blocks), p.chunks);
  int err = 0;
  if constexpr (!BWD) {
    if (scan_has_runs(p, a.T))
      err = own ? launch(gated_scan_fwd_runs_kernel<T, TA, V, V>, runs, block, 0, stream, a)
                : launch(gated_scan_fwd_runs_kernel<T, TA, V, 1>, runs, block, 0, stream, a);
    if (err) return err;
    return own ? launch(gated_scan_fwd_kernel<T, TA, V, V>, grid, block, 0, stream, a)
               : launch(gated_scan_fwd_kernel<T, TA, V, 1>, grid, block, 0, stream, a);
  } else {
    if (scan_has_runs(p, a.T))
      err = own ? launch(gated_scan_bwd_runs_kernel<T, TA, V, V>, runs, block, 0, stream, a)
                : launch(gated_scan_bwd_runs_kernel<T, TA, V, 1>, runs, block, 0, stream, a);
    if (err) return err;
    err = own ? launch(gated_scan_bwd_kernel<T, TA, V, V, false>, grid, block, 0, stream, a)
              : launch(gated_scan_bwd_kernel<T, TA, V, 1, true>, grid, block, 0, stream, a);
    if (err || p.segs == 1) return err;
    const int64_t sums = (int64_t)a.T * a.B * a.G;
    return launch(gated_scan_bwd_finish_kernel<TA>, dim3((unsigned)((sums + 255) / 256)), dim3(256), 0, stream, a, p.segs);
  }
}

static inline int64_t scan_run_floats(const socmx_scan& s, const ScanPlan& p) {
  return scan_has_runs(p, s.T) ? (int64_t)p.chunks * (1 + kScanW) * 2 * s.B * s.D : 0;
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
  const int64_t C = (int64_t)scan->B * scan->D, runs = scan_run_floats(*scan, p);
  *state_floats = (scan->T + kScanU - 1) / kScanU * C;
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
  if (scan_has_runs(p, scan->T) && !workspace) return SOCMX_E_WORKSPACE;
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
  if ((scan_has_runs(p, scan->T) || p.segs > 1) && !workspace) return SOCMX_E_WORKSPACE;
  ScanArgs a = scan_args(*scan, p);
  a.x = x; a.alpha = log_decay; a.state = const_cast<float*>(states); a.dh = dh; a.dht = dh_stride_t; a.dhb = dh_stride_b;
  a.dfinal = dfinal; a.dx = dx; a.dxt = dx_stride_t; a.dxb = dx_stride_b;
  a.dalpha = dlog_decay; a.dat = dgate_stride_t; a.dab = dgate_stride_b; a.dinitial = dinitial;
  a.run = workspace;
  a.part = workspace ? workspace + scan_run_floats(*scan, p) : nullptr;
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
