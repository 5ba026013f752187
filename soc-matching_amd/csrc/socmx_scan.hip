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
// ONE READ.  A step is an affine map, so a run of steps is one: h -> exp(S) h + l with S the sum of its alphas and l its result from zero --
// the same form, applied with the code of a step.  A workgroup owns 64 V channels and a chunk of W U steps, a wave U of them, in registers.
// Every wave forms its run's (S, l); the waves meet in LDS; the workgroup leaves its chunk's (q, l) in memory for the chunks behind it, takes
// those in front of it from there, and its waves walk their steps from the state they find.  So x and alpha are read once and h is
// written once, however few channels there are.
//   Who waits for whom: chunks are dealt out by a ticket in the order of the steps, so a chunk waits only for workgroups that have started
// and that leave their (q, l) without waiting for anybody.  A chunk takes a group's chunks at most, in order; the state at every
// group's first chunk is left by the chunk in front of it, which is the one chain along time.  What is composed with what does not depend on who comes
// first: the same bits on every run.  A word in memory is its own flag: it is set to kEmpty by a launch before this one, written once by one
// 64-bit store, and read until it is something else -- no fence, which would write back the cache of a whole die.  A wait that lasts
// kPolls reads (about a second) ends in NaN: the launch ends whatever happens.
//
// THE BACKWARD is the same from the end.  It rebuilds a wave's U steps of h in f32 from the state that the forward leaves in front of them
// (f32, 1 / U of h) -- h itself, rounded to 16 bits, would put its rounding into dalpha.  A gate shared by several channels: their
// products are summed across the lanes in a fixed order, gates wider than a wave leave one partial sum a wave for another launch.  No
// floating-point atomics.
//
// MEASURED (forward + backward): f32 (65536, 1, 640), a decay each: 112 to 121 us (4.2 to 4.6 TB/s of x, alpha, h and states) + 158 to 168 us (5.1 to 5.4):
// memory, a copy of this size runs at 4.9.  bf16 (4096, 8, 2048), 32 decays a step: 63 us (4.6 TB/s) + 103 us (4.1); rows of 0 to 4096 steps, 55 % of
// them in all, 60 + 95 (3.8, 3.2), of which arithmetic is 20 + 32.  f32 (201, 128, 256), 8 decays: 14 + 21.  Results leave past the caches (5 % less
// than through them).
// Reading x and alpha twice -- once for the runs, once for the steps, in launches of their own -- took 447, 238 and 57 us together.  U = 16 was the
// best among 4, 8, 16; chunks wait for each other 3 to 7 % of the time.  Workgroups that stay and draw their next ticket early hold up
// whoever waits for it: 283 -> 315 us for the first shape.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <utility>

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
  uint64_t* word;                    // (chunks, B D): q and l of every chunk; then (ceil(chunks / group), B D) floats: the state at its first
  float* mark;                       //   chunk; then the ticket (more than one chunk only)
  uint32_t* ticket;
  float* part;                       // (T, B G, segments): partial sums of dalpha (gates wider than a wave only)
  const int32_t* lengths;            // (B,), nullable
  int64_t xt, xb, at, ab, ht, hb, dht, dhb;   // elements between steps / rows of x, alpha, h, dh
  int64_t dxt, dxb, dat, dab;                 // of dx, dalpha
  int T, B, D, G, reverse;
  int chunks, group;                 // every group-th chunk has its state marked (group <= kGroup)
  uint32_t blocks;                   // workgroups a chunk
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

// the gate of a step that leaves the state as it is: of every finite state (an infinite one times it is not left out of the sum), so the steps
// behind a row's length are not applied, and runs of nothing but them (run_apply) leave its product away
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

// Runs of steps: the sum of their alphas (-inf if a gate forgets, whatever the others are), the gate of all of them -- one that forgets only if a
// single one does: a state that is NaN in front of gates whose product is below 2^-126 stays so -- and the run applied to a state.  From a
// state of zero it is its own result, also where the gates' product is beyond f32.
__device__ __forceinline__ float run_join(float s, float t) {
  constexpr float cut = -__builtin_inff();
  return s == cut || t == cut ? cut : s + t;
}
__device__ __forceinline__ float run_gate(float sum) {
  const float q = gate_of(sum);
  return q == 0.f && sum != -__builtin_inff() ? 1.17549435e-38f : q;
}
__device__ __forceinline__ float run_apply(float q, float h, float l) {
  const float v = fmaf(gate_keeps(q), h, fmaf(q, q == kGateKeeps ? 0.f : h, l));
  return h == 0.f || q == 0.f ? l : v;             // (what hangs on h is short: runs are joined one after the other)
}

constexpr int kScanU = 16, kGroup = 16;
constexpr int kPolls = 1 << 20;
constexpr uint64_t kEmpty = ~0ull;
constexpr uint32_t kNoState = ~0u;

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
__device__ __forceinline__ ScanLane scan_lane(const ScanArgs& a, uint32_t block) {
  ScanLane l;
  const int lane = threadIdx.x & 63, per = a.D / a.G;
  l.group = 0; l.seg = 0; l.at = 0; l.lanes = 1; l.first = 1;
  if constexpr (GROUPED) {
    const int wide = per / V;        // lanes of a gate
    if (wide <= 64) {
      const int fit = 64 / wide;
      l.group = (int64_t)block * fit + lane / wide;
      l.at = lane % wide;
      l.lanes = wide;
      l.live = lane / wide < fit && l.group < (int64_t)a.B * a.G;
      l.c = l.at * V;
    } else {
      const int segs = (wide + 63) / 64;
      l.group = block / segs;
      l.seg = block % segs;
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
    l.ch = ((int64_t)block * 64 + lane) * V;
    l.live = l.ch < (int64_t)a.B * a.D;
    if (!l.live) l.ch = 0;
    l.b = (int)(l.ch / a.D);
    l.c = (int)(l.ch % a.D);
    l.gate = l.c / per;
  }
  l.len = a.lengths ? min(max(a.lengths[l.b], 0), a.T) : a.T;      // (a lane without channels walks along with channel 0 and stores nothing)
  return l;
}

// the address of a row's step 0, and the distance from a step to the next one, in the row's direction
template <typename T>
__device__ __forceinline__ T* scan_origin(T* p, const ScanArgs& a, const ScanLane& l, int64_t st, int64_t sb, int c) {
  return p + (int64_t)l.b * sb + c + (a.reverse && l.len > 0 ? (int64_t)(l.len - 1) * st : 0);
}

// What the compiler is not to see through.  It would keep, from one pass over the steps to the next, the sixteen addresses of every array,
// the elements widened to f32 and what is derived from the gates: registers without which twice the waves fit.
template <typename T>
__device__ __forceinline__ void scan_next(T*& p, int64_t d) {
  p += d;
  asm("" : "+v"(p));
}
template <typename T, int V>
__device__ __forceinline__ void scan_forget(reg_vec<T, V>& r) {
  if constexpr (sizeof(T) * V == 8) {
    uint64_t w = __builtin_bit_cast(uint64_t, r);
    asm("" : "+v"(w));
    r = __builtin_bit_cast(reg_vec<T, V>, w);
  } else if constexpr (sizeof(T) * V == 4) {
    uint32_t w = __builtin_bit_cast(uint32_t, r);
    asm("" : "+v"(w));
    r = __builtin_bit_cast(reg_vec<T, V>, w);
  }
}
template <int NA>
__device__ __forceinline__ void scan_forget(float (&q)[kScanU][NA]) {
#pragma unroll
  for (int u = 0; u < kScanU; ++u)
#pragma unroll
    for (int i = 0; i < NA; ++i) asm("" : "+v"(q[u][i]));
}

// U steps from step k0 on, V values each; nothing is read behind the length
template <typename T, int V>
__device__ __forceinline__ void scan_load(reg_vec<T, V> (&out)[kScanU], const T* origin, int64_t d, int k0, int len, bool full) {
  const T* p = origin + (int64_t)k0 * d;
  if (full) {
#pragma unroll
    for (int u = 0; u < kScanU; ++u, scan_next(p, d)) out[u] = load_vec<T, V>(p);
  } else {
#pragma unroll
    for (int u = 0; u < kScanU; ++u, scan_next(p, d))
      if (k0 + u < len) out[u] = load_vec<T, V>(p);
  }
}

template <int... U>
__device__ __forceinline__ void gate_hand(float (&q)[kScanU][1], float g, std::integer_sequence<int, U...>) {
  ((q[U][0] = dpp_move<0x150 + U>(g)), ...);       // (lane U of the row to all of them)
}

// q of U steps and the sum of their alphas (-inf once a gate forgets); whether one of this wave's gates does.  origin: alpha at step 0.
// ROW: the 16 lanes of a row share their gate.  Lane u of a row takes step u -- one load and one gate instead of sixteen -- and hands it to the
// others.
// meanwhile(): what is loaded behind them.
template <typename TA, int NA, bool ROW, typename F>
__device__ __forceinline__ bool scan_gates(float (&q)[kScanU][NA], float (&sum)[NA], const TA* origin, int64_t d, int k0, int len, bool full, F&& meanwhile) {
  bool cut = false;
  if constexpr (ROW) {
    static_assert(NA == 1 && kScanU == 16, "a gate for a row of 16 lanes, a step for each of them");
    const int u = threadIdx.x & 15;
    const bool in = full || k0 + u < len;
    float g = kGateKeeps, s = 0.f;
    TA raw = (TA)0.f;
    if (in) raw = origin[(int64_t)(k0 + u) * d];
    meanwhile();
    if (in) {
      s = (float)raw;
      g = gate_of(s);
      cut = g == 0.f;
    }
    const float any = lanes_sum<16>(cut ? 1.f : 0.f);
    sum[0] = lanes_sum<16>(s);
    if (any > 0.f) sum[0] = -__builtin_inff();
    gate_hand(q, g, std::make_integer_sequence<int, kScanU>{});
  } else {
    reg_vec<TA, NA> raw[kScanU];
    scan_load<TA, NA>(raw, origin, d, k0, len, full);
    meanwhile();
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      bool zero = false;
      sum[i] = 0.f;
#pragma unroll
      for (int u = 0; u < kScanU; ++u) {
        const bool in = full || k0 + u < len;
        const float alpha = raw[u][i];
        q[u][i] = in ? gate_of(alpha) : kGateKeeps;
        sum[i] += in ? alpha : 0.f;
        zero |= q[u][i] == 0.f;
      }
      if (zero) sum[i] = -__builtin_inff();
      cut |= zero;
    }
  }
  return __any(cut);
}

// ---- the chunks in front ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t filled(float v) {              // never the bits that mean empty (one of the patterns of NaN)
  const uint32_t u = __float_as_uint(v);
  return u == kNoState ? 0x7FC00000u : u;
}

__device__ __forceinline__ void leave_word(uint64_t* p, float q, float l) {
  const uint64_t v = (uint64_t)filled(q) | (uint64_t)__float_as_uint(l) << 32;
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void leave_state(float* p, float s) {
  __hip_atomic_store(reinterpret_cast<uint32_t*>(p), filled(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// N words each lane with `need` waits for
template <int N>
__device__ __forceinline__ void take_words(float (&q)[N], float (&l)[N], const uint64_t* p, bool need) {
  uint64_t v[N];
  for (int left = kPolls;; --left) {
    bool missing = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = need ? __hip_atomic_load(const_cast<uint64_t*>(p) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
      missing |= need && v[i] == kEmpty;
    }
    if (!__any(missing) || left == 0) break;
    __builtin_amdgcn_s_sleep(0);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = __uint_as_float((uint32_t)v[i]);        // (kEmpty after kPolls reads: NaN)
    l[i] = __uint_as_float((uint32_t)(v[i] >> 32));
  }
}
__device__ __forceinline__ float take_state(const float* p, bool need) {
  uint32_t v;
  for (int left = kPolls;; --left) {
    v = need ? __hip_atomic_load(reinterpret_cast<uint32_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    if (!__any(need && v == kNoState) || left == 0) break;
    __builtin_amdgcn_s_sleep(0);
  }
  return __uint_as_float(v);
}

__global__ __launch_bounds__(256) void gated_scan_clear_kernel(uint64_t* word, int64_t words, uint32_t* ticket) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < words) word[i] = kEmpty;                 // (two empty states a word in the second part)
  if (i == 0) *ticket = 0;
}

template <int W, int V, int NA>
struct ScanMeet {                                  // where the waves of a workgroup meet
  float q[W][NA][64], sum[W][NA][64], l[W][V][64];       // the waves' runs
  float pq[kGroup - 1][V][64], pl[kGroup - 1][V][64];   // the chunks in front, back to the last marked one
  float in[V][64];                                 // the state in front of (behind) the chunk
  uint32_t ticket;
};

// the number of this workgroup among all of its launch, in the order in which they start
template <int W, int V, int NA>
__device__ __forceinline__ uint32_t scan_ticket(const ScanArgs& a, ScanMeet<W, V, NA>& m) {
  if (a.chunks == 1) return blockIdx.x;
  if (threadIdx.x == 0) m.ticket = atomicAdd(a.ticket, 1u);
  __syncthreads();
  return m.ticket;
}

// The waves' runs (sum, run: this wave's) into the meeting place, and the chunk's (q, l) into memory, for the chunks behind chunk `chunk`
// (counted in the walk's direction).  The first V waves do that, for one of a lane's channels each.  BACK: the waves' order within the chunk
// is the opposite one.
template <bool BACK, int W, int V, int NA>
__device__ __forceinline__ void scan_leave(ScanMeet<W, V, NA>& m, const ScanArgs& a, const ScanLane& l, int chunk, const float (&sum)[NA],
                                           const float (&run)[V], float& chunk_q, float& chunk_l) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    m.q[wave][i][lane] = run_gate(sum[i]);
    m.sum[wave][i][lane] = sum[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) m.l[wave][i][lane] = run[i];
  __syncthreads();
  chunk_q = chunk_l = 0.f;
  if (wave < V) {
    const int gate = NA == 1 ? 0 : wave;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int w = BACK ? W - 1 - k : k;
      chunk_q = run_join(chunk_q, m.sum[w][gate][lane]);
      chunk_l = run_apply(m.q[w][gate][lane], chunk_l, m.l[w][wave][lane]);
    }
    chunk_q = run_gate(chunk_q);
    if (chunk + 1 < a.chunks && (chunk + 1) % a.group != 0 && l.live)
      leave_word(a.word + chunk * ((int64_t)a.B * a.D) + l.ch + wave, chunk_q, chunk_l);
  }
}

// the state in front of the chunk into m.in; first: the state in front of all steps
template <int W, int V, int NA>
__device__ __forceinline__ void scan_take(ScanMeet<W, V, NA>& m, const ScanArgs& a, const ScanLane& l, int chunk, float chunk_q, float chunk_l,
                                          const float* first) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t C = (int64_t)a.B * a.D;
  const int marked = chunk / a.group * a.group;
  for (int j = wave; j < chunk - marked; j += W) {
    float q[V], t[V];
    take_words<V>(q, t, a.word + (marked + j) * C + l.ch, l.live);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      m.pq[j][i][lane] = q[i];
      m.pl[j][i][lane] = t[i];
    }
  }
  float s = 0.f;
  if (wave < V) {
    if (marked > 0) s = take_state(a.mark + marked / a.group * C + l.ch + wave, l.live);
    else if (first && l.live) s = first[l.ch + wave];
  }
  __syncthreads();
  if (wave < V) {
#pragma unroll 4
    for (int j = 0; j < chunk - marked; ++j) s = run_apply(m.pq[j][wave][lane], s, m.pl[j][wave][lane]);
    m.in[wave][lane] = s;
    if (chunk + 1 < a.chunks && (chunk + 1) % a.group == 0 && l.live)
      leave_state(a.mark + (chunk + 1) / a.group * C + l.ch + wave, run_apply(chunk_q, s, chunk_l));
  }
  __syncthreads();
}

// a wave's own state: the chunk's, past the waves in front
template <bool BACK, int W, int V, int NA>
__device__ __forceinline__ void scan_own_state(float (&h)[V], const ScanMeet<W, V, NA>& m) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = m.in[i][lane];
  for (int k = 0; k < (BACK ? W - 1 - wave : wave); ++k) {
    const int w = BACK ? W - 1 - k : k;
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = run_apply(m.q[w][NA == 1 ? 0 : i][lane], h[i], m.l[w][i][lane]);
  }
}

template <typename T, typename TA, int W, int V, int NA, bool ROW>
__global__ __launch_bounds__(64 * W, 4) void gated_scan_fwd_kernel(const ScanArgs a) {
  __shared__ ScanMeet<W, V, NA> meet;
  const uint32_t number = scan_ticket(a, meet);
  const int wave = threadIdx.x >> 6, chunk = number / a.blocks;
  const ScanLane l = scan_lane<V, false>(a, number % a.blocks);
  const int64_t C = (int64_t)a.B * a.D;
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, dh = a.reverse ? -a.ht : a.ht;
  const int k0 = (chunk * W + wave) * kScanU;
  const bool full = __all(k0 + kScanU <= l.len), none = !__any(l.live && k0 < l.len);
  reg_vec<T, V> rx[kScanU];
  float q[kScanU][NA], sum[NA] = {}, h[V];
  bool cut = false;
  if (!none) {
    cut = scan_gates<TA, NA, ROW>(q, sum, scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, NA == 1 ? l.gate : l.c), da, k0, l.len, full, [&] {
      scan_load<T, V>(rx, scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c), dx, k0, l.len, full);
    });
  }
  // the run from zero; the steps themselves afterwards, with the same code
  auto walk = [&](auto CUT, auto FULL, auto&& each) {
#pragma unroll
    for (int u = 0; u < kScanU; ++u) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool in = decltype(FULL)::value || k0 + u < l.len;
        const float g = q[u][NA == 1 ? 0 : i], next = gate_apply<decltype(CUT)::value>(g, gate_keeps(g), h[i], in ? rx[u][i] : 0.f);
        h[i] = in ? next : h[i];
      }
      each(u);
    }
  };
  const bool plain = full && !cut;
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = 0.f;
  if (plain) walk(std::false_type{}, std::true_type{}, [](int) {});
  else if (!none) walk(std::true_type{}, std::false_type{}, [](int) {});
  float chunk_q, chunk_l;
  scan_leave<false>(meet, a, l, chunk, sum, h, chunk_q, chunk_l);
  scan_take(meet, a, l, chunk, chunk_q, chunk_l, a.initial);
  scan_forget<NA>(q);
#pragma unroll
  for (int u = 0; u < kScanU; ++u) scan_forget(rx[u]);
  if (k0 >= a.T) return;
  scan_own_state<false>(h, meet);
  if (a.state && l.live) store_vec<float, V>(a.state + (int64_t)(k0 / kScanU) * C + l.ch, h);
  T* h0 = scan_origin(static_cast<T*>(a.h), a, l, a.ht, a.hb, l.c) + (int64_t)k0 * dh;
  T* pad = static_cast<T*>(a.h) + (int64_t)l.b * a.hb + l.c + (int64_t)k0 * a.ht;        // steps behind the length lie at their own index
  if (plain) {
    walk(std::false_type{}, std::true_type{}, [&](int) {
      if (l.live) stream_vec<T, V>(h0, h);
      scan_next(h0, dh);
    });
  } else if (none) {
    const float zero[V] = {};
    for (int u = 0; u < kScanU && k0 + u < a.T; ++u, pad += a.ht)
      if (l.live) stream_vec<T, V>(pad, zero);
  } else {
    walk(std::true_type{}, std::false_type{}, [&](int u) {
      const float zero[V] = {};
      if (l.live && k0 + u < l.len) stream_vec<T, V>(h0, h);
      else if (l.live && k0 + u < a.T) stream_vec<T, V>(pad, zero);
      scan_next(h0, dh);
      scan_next(pad, a.ht);
    });
  }
  if (a.final && k0 + kScanU >= a.T && l.live) store_vec<float, V>(a.final + l.ch, h);
}

// The sums of N values over a gate's lanes of this wave, in the lane `at` = 0.  A power of two of them lies on its own boundary.
template <int N>
__device__ __forceinline__ void gate_lanes_sum(float (&v)[N], int at, int lanes) {
  auto all = [&](auto L) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lanes_sum<decltype(L)::value>(v[k]);
  };
  switch (lanes) {
    case 1: return;
    case 2: return all(std::integral_constant<int, 2>{});
    case 4: return all(std::integral_constant<int, 4>{});
    case 8: return all(std::integral_constant<int, 8>{});
    case 16: return all(std::integral_constant<int, 16>{});
    case 32: return all(std::integral_constant<int, 32>{});
    case 64: return all(std::integral_constant<int, 64>{});
    default: break;
  }
  int off = 1;
  while (off * 2 < lanes) off *= 2;
  for (; off > 0; off /= 2) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float other = __shfl_down(v[k], off, 64);
      if (at + off < lanes) v[k] += other;
    }
  }
}

// ROW: the sums of 16 values over a gate's lanes (a multiple of 16), lane u of a row ending with the u-th.  In four steps a lane and its mirror
// image in the row, in half of it, and so on each keep one half of the values and give the other away.
__device__ __forceinline__ float gate_row_sums(const float (&v)[16], int lanes) {
  const int lane = threadIdx.x & 15;
  float a[8], b[4], c[2];
#pragma unroll
  for (int k = 0; k < 8; ++k) a[k] = (lane & 8 ? v[k + 8] : v[k]) + dpp_move<0x140>(lane & 8 ? v[k] : v[k + 8]);
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = (lane & 4 ? a[k + 4] : a[k]) + dpp_move<0x141>(lane & 4 ? a[k] : a[k + 4]);
#pragma unroll
  for (int k = 0; k < 2; ++k) c[k] = (lane & 2 ? b[k + 2] : b[k]) + dpp_move<0x1B>(lane & 2 ? b[k] : b[k + 2]);
  float s = (lane & 1 ? c[1] : c[0]) + dpp_move<0xB1>(lane & 1 ? c[0] : c[1]);
  // the rows of a gate, in order: the first one of each gate ends with the sum
  const float s1 = __shfl_down(s, 16, 64), s2 = __shfl_down(s, 32, 64), s3 = __shfl_down(s, 48, 64);
  if (lanes > 16) s += s1;
  if (lanes > 32) s += s2;
  if (lanes > 48) s += s3;
  return s;
}

// GROUPED: a gate has several channels (NA = 1); otherwise every channel has its own (NA = V).  Chunks are counted from the end.
// 8 bytes a lane and step need 180 to 250 registers, 2 waves a SIMD (3 of them, spilling: 131 -> 163 us); less fits 128 with a
// step's a_k h_{k-1} kept for half of the steps at a time.
template <typename T, typename TA, int W, int V, int NA, bool GROUPED, bool ROW>
__global__ __launch_bounds__(64 * W, sizeof(T) * V == 8 ? 2 : 4) void gated_scan_bwd_kernel(const ScanArgs a) {
  __shared__ ScanMeet<W, V, NA> meet;
  const uint32_t number = scan_ticket(a, meet);
  const int wave = threadIdx.x >> 6, chunk = number / a.blocks;
  const ScanLane l = scan_lane<V, GROUPED>(a, number % a.blocks);
  const int64_t C = (int64_t)a.B * a.D;
  const int64_t dx = a.reverse ? -a.xt : a.xt, da = a.reverse ? -a.at : a.at, dd = a.reverse ? -a.dht : a.dht;
  const int64_t ddx = a.reverse ? -a.dxt : a.dxt, dda = a.reverse ? -a.dat : a.dat;
  const int gate = NA == 1 ? l.gate : l.c;
  const int k0 = ((a.chunks - 1 - chunk) * W + wave) * kScanU;
  const bool full = __all(k0 + kScanU <= l.len), none = !__any(l.live && k0 < l.len), begun = k0 < a.T;
  reg_vec<T, V> rx[kScanU], rd[kScanU];
  reg_vec<float, V> rs;
  float q[kScanU][NA], sum[NA] = {}, g[V];
  bool cut = false;
#pragma unroll
  for (int u = 0; u < kScanU; ++u) rd[u] = reg_vec<T, V>{};
  if (!none) {
    cut = scan_gates<TA, NA, ROW>(q, sum, scan_origin(static_cast<const TA*>(a.alpha), a, l, a.at, a.ab, gate), da, k0, l.len, full, [&] {
      if (a.dh) scan_load<T, V>(rd, scan_origin(static_cast<const T*>(a.dh), a, l, a.dht, a.dhb, l.c), dd, k0, l.len, full);
    });
  }
  const bool plain = full && !cut;
  auto value = [&](const reg_vec<T, V>& r, int u, int i, bool all) { return all || k0 + u < l.len ? r[i] : 0.f; };
  auto back = [&](auto CUT, auto FULL) {
#pragma unroll
    for (int u = kScanU - 1; u >= 0; --u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float c = q[u][NA == 1 ? 0 : i], d = value(rd[u], u, i, decltype(FULL)::value);
        const float next = gate_times<decltype(CUT)::value>(c, gate_keeps(c), g[i] + d);
        g[i] = decltype(FULL)::value || k0 + u < l.len ? next : g[i];
      }
  };
#pragma unroll
  for (int i = 0; i < V; ++i) g[i] = 0.f;
  if (plain) back(std::false_type{}, std::true_type{});
  else if (!none) back(std::true_type{}, std::false_type{});
  float chunk_q, chunk_l;
  scan_leave<true>(meet, a, l, chunk, sum, g, chunk_q, chunk_l);
  // (x and the state are needed from here on: their way from memory is the wait for the other chunks)
  if (!none) scan_load<T, V>(rx, scan_origin(static_cast<const T*>(a.x), a, l, a.xt, a.xb, l.c), dx, k0, l.len, full);
  if (begun) rs = load_vec<float, V>(a.state + (int64_t)(k0 / kScanU) * C + l.ch);
  scan_take(meet, a, l, chunk, chunk_q, chunk_l, a.dfinal);
  scan_forget<NA>(q);
#pragma unroll
  for (int u = 0; u < kScanU; ++u) scan_forget(rd[u]);
  if (!begun) return;
  scan_own_state<true>(g, meet);
  const int segs = GROUPED ? (a.D / a.G / V + 63) / 64 : 1;
  TA* const alpha0 = scan_origin(static_cast<TA*>(a.dalpha), a, l, a.dat, a.dab, gate);
  TA* const alpha_pad = static_cast<TA*>(a.dalpha) + (int64_t)l.b * a.dab + gate;
  // the gradient of the gate of step k, where the row has it
  auto put_gate = [&](int k, float v) {
    if (!l.live || k >= a.T) return;
    const bool in = k < l.len;
    if (segs > 1) a.part[((int64_t)(in && a.reverse ? l.len - 1 - k : k) * a.B * a.G + l.group) * segs + l.seg] = v;
    else if (in) alpha0[(int64_t)k * dda] = (TA)v;
    else alpha_pad[(int64_t)k * a.dat] = (TA)v;
  };
  if (none) {
    const float zero[V] = {}, none_of[NA] = {};
    T* padx = static_cast<T*>(a.dx) + (int64_t)l.b * a.dxb + l.c;
    for (int k = k0; k < k0 + kScanU && k < a.T; ++k) {
      if (l.live) stream_vec<T, V>(padx + (int64_t)k * a.dxt, zero);
      if constexpr (GROUPED) {
        if (l.first) put_gate(k, 0.f);
      } else {
        if (l.live) stream_vec<TA, NA>(alpha_pad + (int64_t)k * a.dat, none_of);
      }
    }
    if (a.dinitial && k0 == 0 && l.live) store_vec<float, V>(a.dinitial + l.ch, g);
    return;
  }
  T* gx0 = scan_origin(static_cast<T*>(a.dx), a, l, a.dxt, a.dxb, l.c) + (int64_t)(k0 + kScanU - 1) * ddx;
  T* padx = static_cast<T*>(a.dx) + (int64_t)l.b * a.dxb + l.c + (int64_t)(k0 + kScanU - 1) * a.dxt;
  TA* ga0 = alpha0 + (int64_t)(k0 + kScanU - 1) * dda;
  TA* pada = alpha_pad + (int64_t)(k0 + kScanU - 1) * a.dat;
  float gate_grad[GROUPED ? kScanU : 1];
  auto walk = [&](auto CUT, auto FULL) {
    constexpr bool cuts = decltype(CUT)::value, all = decltype(FULL)::value;
    // (the later half first: the walk to it passes the earlier one)
    constexpr int HALF = sizeof(T) * V == 8 ? kScanU : kScanU / 2;
#pragma unroll
    for (int part = kScanU / HALF - 1; part >= 0; --part) {
    float p[HALF][V], h[V];              // p: a_k h_{k-1}
    if (part == 0 && HALF < kScanU) {
      scan_forget<NA>(q);
#pragma unroll
      for (int u = 0; u < HALF; ++u) scan_forget(rx[u]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = rs[i];
#pragma unroll
    for (int u = 0; u < (part + 1) * HALF; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float c = q[u][NA == 1 ? 0 : i], before = gate_times<cuts>(c, gate_keeps(c), h[i]);
        if (u >= part * HALF) p[u - part * HALF][i] = before;
        h[i] = before + value(rx[u], u, i, all);
      }
#pragma unroll
    for (int u = (part + 1) * HALF - 1; u >= part * HALF; --u) {
      const int k = k0 + u;
      const bool in = l.live && (all || k < l.len), behind = !all && l.live && !in && k < a.T;
      float gx[V], galpha[NA] = {};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float c = q[u][NA == 1 ? 0 : i];
        gx[i] = g[i] + value(rd[u], u, i, all);
        galpha[NA == 1 ? 0 : i] += p[u - part * HALF][i] * gx[i];
        const float next = gate_times<cuts>(c, gate_keeps(c), gx[i]);
        g[i] = all || k < l.len ? next : g[i];
      }
      if (in) {
        stream_vec<T, V>(gx0, gx);
      } else if (behind) {
        const float zero[V] = {};
        stream_vec<T, V>(padx, zero);
      }
      scan_next(gx0, -ddx);
      if constexpr (!all) scan_next(padx, -a.dxt);
      if constexpr (GROUPED) {
        gate_grad[u] = in ? galpha[0] : 0.f;
      } else {
        if (in) {
          stream_vec<TA, NA>(ga0, galpha);
        } else if (behind) {
          const float zero[NA] = {};
          stream_vec<TA, NA>(pada, zero);
        }
        scan_next(ga0, -dda);
        if constexpr (!all) scan_next(pada, -a.dat);
      }
    }
    }
  };
  if (plain) walk(std::false_type{}, std::true_type{}); else walk(std::true_type{}, std::false_type{});
  if constexpr (ROW) {
    const float v = gate_row_sums(gate_grad, l.lanes);
    if (l.at < 16) put_gate(k0 + (threadIdx.x & 15), v);
  } else if constexpr (GROUPED) {
    gate_lanes_sum<kScanU>(gate_grad, l.at, l.lanes);
    if (l.first) {
#pragma unroll
      for (int u = 0; u < kScanU; ++u) put_gate(k0 + u, gate_grad[u]);
    }
  }
  if (a.dinitial && k0 == 0 && l.live) store_vec<float, V>(a.dinitial + l.ch, g);
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
  const float q = gate_of((float)alpha[b * ab + c / per]), v = gate_apply<true>(q, gate_keeps(q), *s, (float)x[b * xb + c]);
  *s = v;
  h[i] = (T)v;
}

// ---- launches ------------------------------------------------------------------------------------------------------------------
struct ScanPlan {
  int W, V, chunks, group, segs;
  int64_t blocks, words;               // workgroups a chunk; 64-bit words of workspace for the chunks, the ticket's included
};

// V channels a lane: up to 8 bytes of x and of gates of their own a step, where they divide the channels of a row (of a gate): the forward of
// bf16 (4096, 8, 2048), 32 decays, takes 70 us with 4 channels, 88 with 2 and 130 with 1.  One in the backward with gates of their own, two of
// which spill: 104 us for 113 at bf16 (8192, 4, 1024).
// W waves a workgroup: 16 in the forward, so that fewer chunks wait for each other -- 80 -> 70 us for the shape above, 40 -> 31 for bf16
// (30000, 1, 100) with one decay -- but 8 for f32 channels with gates of their own, which fill the memory's time as it is ((65536, 1, 640): 116
// us for 128), and 8 in the backward, whose registers 16 waves do not have (127 us for 232).
// group: a chunk takes up to group - 1 chunks and one state.  Where few workgroups make a chunk many chunks are under way, and the chain of
// states is what they wait for: (30000, 1, 100) backward 44 us with 16, 57 with 8; with many workgroups a chunk shorter takes are better: the first
// shape's backward 123 us with 8, 127 with 16.
static ScanPlan scan_plan(const socmx_scan& s, bool bwd) {
  ScanPlan p;
  const int64_t C = (int64_t)s.B * s.D;
  const int per = s.D / s.G;
  p.V = 1;
  const int bytes = (s.type == SOCMX_F32 ? 4 : 2) + (per > 1 ? 0 : s.gate_type == SOCMX_F32 ? 4 : 2);
  for (int v = 4; v > 1; v /= 2)
    if (bytes * v <= 8 && s.D % v == 0 && (per == 1 ? !bwd : per % v == 0)) { p.V = v; break; }
  p.W = bwd || (per == 1 && s.type == SOCMX_F32) ? 8 : 16;
  p.blocks = (C + 64 * p.V - 1) / (64 * p.V);
  p.segs = 1;
  if (bwd && per > 1) {
    const int wide = per / p.V;
    p.segs = wide <= 64 ? 1 : (wide + 63) / 64;
    const int64_t gates = (int64_t)s.B * s.G;
    p.blocks = wide <= 64 ? (gates + 64 / wide - 1) / (64 / wide) : gates * p.segs;
  }
  p.chunks = (s.T + p.W * kScanU - 1) / (p.W * kScanU);
  p.group = p.blocks >= 16 ? kGroup / 2 : kGroup;
  p.words = p.chunks > 1 ? p.chunks * C + ((p.chunks + p.group - 1) / p.group * C + 1) / 2 + 1 : 0;
  return p;
}
// (a launch counts its threads in 32 bits)
static bool scan_fits(const ScanPlan& p) { return p.blocks * p.chunks <= UINT32_MAX / (64 * p.W); }

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
  a.chunks = p.chunks; a.group = p.group; a.blocks = (uint32_t)p.blocks;
  return a;
}

template <typename T, typename TA, int V, bool BWD>
static int launch_scan(ScanArgs a, const ScanPlan& p, void* workspace, void* stream) {
  const bool own = a.G == a.D, row = !own && a.D / a.G % (16 * V) == 0;      // (whole rows of lanes share a gate)
  if (p.chunks > 1) {
    const int64_t C = (int64_t)a.B * a.D;
    a.word = static_cast<uint64_t*>(workspace);
    a.mark = reinterpret_cast<float*>(a.word + p.chunks * C);
    a.ticket = reinterpret_cast<uint32_t*>(a.word + p.words - 1);
    if (const int err = launch(gated_scan_clear_kernel, dim3((unsigned)((p.words - 1 + 255) / 256)), dim3(256), 0, stream, a.word, p.words - 1, a.ticket))
      return err;
  }
  const dim3 grid((unsigned)(p.blocks * p.chunks)), block(64 * p.W);
  int err = SOCMX_E_DIM;               // (the forms that scan_plan never asks for are not compiled)
  // (a gate of 16 V channels leaves V at its widest)
  constexpr bool can_own = BWD ? V == 1 : (sizeof(T) + sizeof(TA)) * V <= 8, can_share = sizeof(T) * V <= 8, can_row = sizeof(T) * V == 8;
  if constexpr (!BWD) {
    if constexpr (can_own)
      if (own) return launch(gated_scan_fwd_kernel<T, TA, sizeof(T) == 4 ? 8 : 16, V, V, false>, grid, block, 0, stream, a);
    if constexpr (can_row)
      if (row) return launch(gated_scan_fwd_kernel<T, TA, 16, V, 1, true>, grid, block, 0, stream, a);
    if constexpr (can_share)
      if (!own && !row) return launch(gated_scan_fwd_kernel<T, TA, 16, V, 1, false>, grid, block, 0, stream, a);
    return err;
  } else {
    if constexpr (can_own)
      if (own) err = launch(gated_scan_bwd_kernel<T, TA, 8, V, V, false, false>, grid, block, 0, stream, a);
    if constexpr (can_row)
      if (row) err = launch(gated_scan_bwd_kernel<T, TA, 8, V, 1, true, true>, grid, block, 0, stream, a);
    if constexpr (can_share)
      if (!own && !row) err = launch(gated_scan_bwd_kernel<T, TA, 8, V, 1, true, false>, grid, block, 0, stream, a);
    if (err || p.segs == 1) return err;
    const int64_t sums = (int64_t)a.T * a.B * a.G;
    return launch(gated_scan_bwd_finish_kernel<TA>, dim3((unsigned)((sums + 255) / 256)), dim3(256), 0, stream, a, p.segs);
  }
}

template <typename T, typename TA, bool BWD>
static int launch_scan_v(const ScanArgs& a, const ScanPlan& p, void* ws, void* stream) {
  if (p.V == 4) return launch_scan<T, TA, 4, BWD>(a, p, ws, stream);
  if (p.V == 2) return launch_scan<T, TA, 2, BWD>(a, p, ws, stream);
  return launch_scan<T, TA, 1, BWD>(a, p, ws, stream);
}

template <bool BWD>
static int dispatch_scan(const socmx_scan& s, const ScanArgs& a, const ScanPlan& p, void* ws, void* stream) {
  const bool wide = s.gate_type == SOCMX_F32;
  if (s.type == SOCMX_F32) return launch_scan_v<float, float, BWD>(a, p, ws, stream);
  if (s.type == SOCMX_BF16) return wide ? launch_scan_v<bf16_t, float, BWD>(a, p, ws, stream) : launch_scan_v<bf16_t, bf16_t, BWD>(a, p, ws, stream);
  return wide ? launch_scan_v<f16_t, float, BWD>(a, p, ws, stream) : launch_scan_v<f16_t, f16_t, BWD>(a, p, ws, stream);
}

}  // namespace socmx

using namespace socmx;

extern "C" int socmx_gated_scan_sizes(const socmx_scan* scan, int64_t* state_floats, int64_t* fwd_workspace_floats,
                                      int64_t* bwd_workspace_floats) {
  if (const int bad = scan_check(scan)) return bad;
  if (!state_floats || !fwd_workspace_floats || !bwd_workspace_floats) return SOCMX_E_NULL;
  const ScanPlan f = scan_plan(*scan, false), b = scan_plan(*scan, true);
  if (!scan_fits(f) || !scan_fits(b)) return SOCMX_E_DIM;
  const int64_t C = (int64_t)scan->B * scan->D;
  *state_floats = (scan->T + kScanU - 1) / kScanU * C;
  *fwd_workspace_floats = 2 * f.words;
  *bwd_workspace_floats = 2 * b.words + (b.segs > 1 ? (int64_t)scan->T * scan->B * scan->G * b.segs : 0);
  return 0;
}

extern "C" int socmx_gated_scan_fwd(const socmx_scan* scan, const void* x, const void* log_decay, const float* initial, void* h,
                                    int64_t h_stride_t, int64_t h_stride_b, float* final_state, float* states, float* workspace,
                                    socmx_stream_t stream) {
  if (const int bad = scan_check(scan)) return bad;
  if (!x || !log_decay || !h) return SOCMX_E_NULL;
  const ScanPlan p = scan_plan(*scan, false);
  if (!scan_fits(p)) return SOCMX_E_DIM;
  if (p.chunks > 1 && (!workspace || (uintptr_t)workspace % 8)) return SOCMX_E_WORKSPACE;
  ScanArgs a = scan_args(*scan, p);
  a.x = x; a.alpha = log_decay; a.initial = initial; a.h = h; a.ht = h_stride_t; a.hb = h_stride_b;
  a.final = final_state; a.state = states;
  return dispatch_scan<false>(*scan, a, p, workspace, stream);
}

extern "C" int socmx_gated_scan_bwd(const socmx_scan* scan, const void* x, const void* log_decay, const float* states, const void* dh,
                                    int64_t dh_stride_t, int64_t dh_stride_b, const float* dfinal, void* dx, int64_t dx_stride_t,
                                    int64_t dx_stride_b, void* dlog_decay, int64_t dgate_stride_t, int64_t dgate_stride_b,
                                    float* dinitial, float* workspace, socmx_stream_t stream) {
  if (const int bad = scan_check(scan)) return bad;
  if (!x || !log_decay || !states || !dx || !dlog_decay) return SOCMX_E_NULL;
  const ScanPlan p = scan_plan(*scan, true);
  if (!scan_fits(p)) return SOCMX_E_DIM;
  if ((p.chunks > 1 || p.segs > 1) && (!workspace || (uintptr_t)workspace % 8)) return SOCMX_E_WORKSPACE;
  ScanArgs a = scan_args(*scan, p);
  a.x = x; a.alpha = log_decay; a.state = const_cast<float*>(states); a.dh = dh; a.dht = dh_stride_t; a.dhb = dh_stride_b;
  a.dfinal = dfinal; a.dx = dx; a.dxt = dx_stride_t; a.dxb = dx_stride_b;
  a.dalpha = dlog_decay; a.dat = dgate_stride_t; a.dab = dgate_stride_b; a.dinitial = dinitial;
  a.part = workspace ? workspace + 2 * p.words : nullptr;
  return dispatch_scan<true>(*scan, a, p, workspace, stream);
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
