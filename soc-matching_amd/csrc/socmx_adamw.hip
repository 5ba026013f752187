// socmx_adamw.hip -- AdamW over many tensors at once, states in 32 or in 8 bits, gfx950.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: with f32 weights 28 bytes an element in 32 bits, 16 in 8 bits.  A workgroup takes 4096 elements of one tensor; the
// tensors' addresses travel in the kernel's arguments (48 tensors a launch), so a call needs no table in device memory and can be
// captured.  Step counts stay on the device: a first launch advances them and forms the bias corrections, in 64 bits.
//
// STATES IN 8 BITS, per block of 256 elements of a tensor, with two f32 scales:  m = S_m c |c| / 127^2 (c in -127..127, S_m = max |m|),
// v = S_v (c / 255)^4 (c in 0..255, S_v = max v).  The levels crowd towards zero as the values do: 1.6 % of the block's maximum
// apart at the top for m and for sqrt(v), 2^-14 and 2^-16 of it the smallest.  An average with weight 1 - b2 = 0.001 moves by less
// than half a level a step, so rounding to the nearest one would freeze it: a state goes to the level above with the probability
// of its place between the two -- unbiased, so that the average keeps its mean -- where the "probability" is a 32-bit mix of the
// element's index and the step: the same on every run, and no random numbers to carry.  Which level it is hangs on the last digits,
// so the states are formed in 64 bits (full rate on this chip), every operation rounded by itself in the order written here: with
// decays like 9/10 a maximum lies exactly between two f32 as often as one time in ten, and a fused product would decide otherwise
// than the same formula elsewhere.  A positive v never becomes 0: eps alone would divide m.
// The weight's update uses m and v as they are before they are rounded.  A block with a value that is not finite gets a NaN scale.
//
// MEASURED, 96 M elements: 32 bits, f32 weights 519 us in 24 tensors (5.2 TB/s) and 547 in 100 at odd offsets (4.9, the rate of a copy of this size),
// bf16 404 (5.2), with f32 masters 513 (5.2).  8 bits: f32 326 to 356, bf16 298 to 327, with masters 337 to 391 (4.6 to 3.9 TB/s; a copy of as many
// bytes 314): arithmetic, 118 instructions an element, issues for 285 us of it, bf16 without masters moves its bytes in 190.  Their decoded
// values 161 us (6.0 TB/s, most of it stores).  Stores past the caches cost 4 %.  18 tensors, 171 k elements: 6.4 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/socmx.h"
#include "socmx_launch.h"
#include "socmx_vec.h"

namespace socmx {

constexpr int kAdamwTensors = 48, kAdamwChunk = 4096, kAdamwBlock = 256, kAdamwCounts = 256;

struct AdamwTensor {
  void* p;
  const void* g;
  void *m, *v;
  float* scale;
  float* master;
  int64_t n;
};

struct AdamwArgs {
  AdamwTensor tensor[kAdamwTensors];
  int32_t first[kAdamwTensors + 1];  // the first workgroup of every tensor
  int32_t count;
  const float* correction;           // (count, 4): lr / (1 - b1^t), 1 / sqrt(1 - b2^t), t (as an integer), unused
  double b1, b2;
  float decay, eps;                  // decay: lr wd
};

struct AdamwValuesArgs {
  const void* m[kAdamwTensors];
  const void* v[kAdamwTensors];
  const float* scale[kAdamwTensors];
  float* out_m[kAdamwTensors];
  float* out_v[kAdamwTensors];
  int64_t n[kAdamwTensors];
  int32_t first[kAdamwTensors + 1];
  int32_t count;
};

// the tensor whose workgroups hold `block` (of several that begin there the last one: the others are empty)
__device__ __forceinline__ int adamw_tensor(const int32_t* first, int count, int block) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= block) lo = mid; else hi = mid;
  }
  return lo;
}

// the step counts, next to each other in memory, or each where it lies
struct AdamwSteps {
  float* at;
  __device__ __forceinline__ float* operator[](int i) const { return at + i; }
};
struct AdamwCounts {
  float* at[kAdamwCounts];
  __device__ __forceinline__ float* operator[](int i) const { return at[i]; }
};

// 1 - b^t in 64 bits, without cancellation
template <typename Steps>
__global__ __launch_bounds__(64) void adamw_begin_kernel(const Steps steps, int n, double log_b1, double log_b2, double lr, float* correction) {
  const int i = blockIdx.x * 64 + threadIdx.x;
  if (i >= n) return;
  const float t = *steps[i] + 1.f;
  *steps[i] = t;
  correction[4 * i] = (float)(lr / -expm1((double)t * log_b1));
  correction[4 * i + 1] = (float)(1.0 / sqrt(-expm1((double)t * log_b2)));
  correction[4 * i + 2] = __uint_as_float((uint32_t)t);
}

__device__ __forceinline__ bool adamw_careful(float eps) { return eps < 1e-10f; }

// The hardware's root and reciprocal, each within one step of f32: two of the update's two dozen roundings.  The root takes numbers below
// 2^-126 for 0.  It is off by 2^-63 then, times 32 for the first steps of a decay of 0.999: nothing beside an eps of 1e-10; with less (careful), small
// numbers are moved up by 2^64 and their root down by 2^-32 (for every eps: 405 us instead of 385 for 96 M 8-bit elements).
__device__ __forceinline__ float adamw_weight(float p, float m, float v, float size, float root, float decay, float eps, bool careful) {
  float deviation;
  if (careful) {
    const bool small = v < 0x1p-100f;
    deviation = __builtin_amdgcn_sqrtf(v * (small ? 0x1p64f : 1.f)) * (small ? 0x1p-32f : 1.f);
  } else {
    deviation = __builtin_amdgcn_sqrtf(v);
  }
  // (What is taken off is formed first: a factor 1 - lr wd in f32 would be off by up to 2^-25, a fifth of a decay of 1e-7 and all of a smaller
  // one.  An infinite weight stays one.)
  const float held = __builtin_amdgcn_fmed3f(p, -3.40282347e38f, 3.40282347e38f);
  float w = p - fmaf(held, decay, size * m * __builtin_amdgcn_rcpf(deviation * root + eps));
  asm("" : "+v"(w));      // a float32 from here on: a 16-bit weight is its rounding, not a second result of one mixed instruction
  return w;
}

template <typename T>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwArgs a) {
  const int k = adamw_tensor(a.first, a.count, blockIdx.x);
  const AdamwTensor t = a.tensor[k];
  const float size = a.correction[4 * k], root = a.correction[4 * k + 1];
  const float b1 = (float)a.b1, c1 = (float)(1.0 - a.b1), b2 = (float)a.b2, c2 = (float)(1.0 - a.b2);
  const int64_t begin = (int64_t)(blockIdx.x - a.first[k]) * kAdamwChunk;
#pragma unroll
  for (int r = 0; r < kAdamwChunk / 1024; ++r) {
    const int64_t i = begin + r * 1024 + threadIdx.x * 4;
    if (i >= t.n) return;
    const int have = (int)std::min<int64_t>(4, t.n - i);
    const reg_vec<T, 4> g = load_vec<T, 4>(static_cast<const T*>(t.g) + i, have);
    const reg_vec<float, 4> m0 = load_vec<float, 4>(static_cast<float*>(t.m) + i, have), v0 = load_vec<float, 4>(static_cast<float*>(t.v) + i, have);
    float p[4], m[4], v[4];
    if (t.master) {
      const reg_vec<float, 4> w = load_vec<float, 4>(t.master + i, have);
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = w[e];
    } else {
      const reg_vec<T, 4> w = load_vec<T, 4>(static_cast<T*>(t.p) + i, have);
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = w[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = b1 * m0[e] + c1 * g[e];
      v[e] = b2 * v0[e] + c2 * (g[e] * g[e]);
      p[e] = adamw_weight(p[e], m[e], v[e], size, root, a.decay, a.eps, adamw_careful(a.eps));
    }
    store_vec<float, 4>(static_cast<float*>(t.m) + i, m, have);
    store_vec<float, 4>(static_cast<float*>(t.v) + i, v, have);
    store_vec<T, 4>(static_cast<T*>(t.p) + i, p, have);
    if (t.master) store_vec<float, 4>(t.master + i, p, have);
  }
}

// two thresholds in (0, 1) from an element's place in its tensor and the step
__device__ __forceinline__ uint32_t adamw_mix(uint32_t i, uint32_t step) {
  uint32_t z = i * 0x9E3779B1u + step * 0xBB67AE85u;      // (odd 32-bit fractions of the golden ratio, sqrt(3) and sqrt(2))
  z ^= z >> 16;
  z *= 0x6A09E667u;
  z ^= z >> 15;
  z *= 0x9E3779B1u;
  z ^= z >> 16;
  return z;
}

// what the scales of 8-bit states are multiplied with when their codes are read, and divided into when codes are formed
constexpr double kTopM = 127.0 * 127.0, kTopV = 255.0 * 255.0 * 255.0 * 255.0;

// the largest of 64 lanes' bit patterns: for magnitudes this is the largest value, and NaN above infinity above all others
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t x) {
  auto dpp = [](uint32_t v, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, true); };
  x = std::max(x, dpp(x, std::integral_constant<int, 0xB1>{}));     // quad_perm [1,0,3,2]
  x = std::max(x, dpp(x, std::integral_constant<int, 0x4E>{}));     // quad_perm [2,3,0,1]
  x = std::max(x, dpp(x, std::integral_constant<int, 0x141>{}));    // mirror of 8 lanes
  x = std::max(x, dpp(x, std::integral_constant<int, 0x140>{}));    // mirror of 16 lanes
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);       // the odd rows of 16 lanes, the even ones
  x = std::max(rows[0], rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return std::max(halves[0], halves[1]);
}

__device__ __forceinline__ double wave_lane(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// a block's scale: its maximum, or NaN where that is not finite
__device__ __forceinline__ float adamw_scale(uint32_t bits) { return bits >= 0x7F800000u ? __builtin_nanf("") : __uint_as_float(bits); }

// A code is c or c + 1 with c^n <= y < (c + 1)^n, the upper one where y - c^n > u ((c + 1)^n - c^n), u = (2 k + 1) / 2^17.  The f32 root,
// taken a little low, gives c or the level below it: the test is made there and once more a level up, and the code is that level and
// one for each test that holds -- the same code either way, with no case to tell apart.  `half`: k.
constexpr float kRootLow = 1.f - 4.8e-7f;                           // (four steps of f32; root and conversion are within two)

// The square of a value that fits 16 bits.  (One full-rate instruction.  The compiler takes the quarter-rate one of 32 bits instead wherever
// it sees that only low bits are used.)
__device__ __forceinline__ uint32_t square_small(uint32_t a) {
  uint32_t r;
  asm("v_mul_u32_u24_e32 %0, %1, %1" : "=v"(r) : "v"(a));
  return r;
}

// (a product of values that fit 24 bits is one full-rate instruction, which looks at no other bits)
__device__ __forceinline__ uint32_t mul_small(uint32_t a, uint32_t b) {
  return (a & 0xFFFFFFu) * (b & 0xFFFFFFu);
}

// y = |m| / S 127^2.  In whole numbers: 2^17 y, rounded up, is above a whole threshold exactly where y is.
__device__ __forceinline__ int adamw_code_m(double y_scaled, uint32_t half) {
  const uint32_t y = (uint32_t)__builtin_ceil(y_scaled);            // at most 2^17 127^2 and a bit: below 2^31
  const uint32_t c = (uint32_t)(__builtin_amdgcn_sqrtf((float)y) * (0.00276213586400995125f * kRootLow));      // 2^-8.5
  const uint32_t rest = y - (square_small(c) << 17), gap = 2 * c + 1, odd = 2 * half + 1, first = mul_small(odd, gap);
  const uint32_t second = (gap << 17) + first + 2 * odd;            // the gap, and u of the next one, which is 2 wider
  return std::min((int)(c + (rest > first) + (rest > second)), 127);
}

// y = v / S 255^4: differences of fourth powers need 64 bits, which hold every term exactly.  Everything times 2^17, as above
__device__ __forceinline__ int adamw_code_v(double y_scaled, uint32_t half) {
#pragma clang fp contract(off)
  const uint32_t c = (uint32_t)(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)y_scaled)) * (0.0525560259536012f * kRootLow));      // 2^-4.25; at most 254
  const uint32_t c2 = square_small(c), d2 = c2 + 2 * c + 1, e2 = d2 + 2 * c + 3;
  const uint32_t c4 = mul_small(c2, c2), d4 = mul_small(d2, d2), e4 = mul_small(e2, e2);    // (256^4 wraps to 0, its difference does not)
  const double odd = (double)(2 * half + 1), rest = __builtin_fma(-131072.0, (double)c4, y_scaled), gap = (double)(d4 - c4);
  return std::min((int)(c + (rest > odd * gap) + (rest > __builtin_fma(odd, (double)(e4 - d4), gap * 131072.0))), 255);
}

template <typename T>
struct Adamw8Block {                 // what a lane needs of its four elements
  reg_vec<T, 4> g, p16;
  reg_vec<float, 4> p32;
  uint32_t cm, cv;
  float sm, sv;
};
typedef uint32_t packed_codes __attribute__((aligned(1)));

// `have` of the four elements from `i` on (4 and nothing else where FULL)
template <typename T, bool MASTER, bool FULL>
__device__ __forceinline__ Adamw8Block<T> adamw8_load(const AdamwTensor& t, int64_t block, int64_t i, int have) {
  Adamw8Block<T> b;
  if (FULL) have = 4;
  const int64_t at = FULL || have ? i : 0;
  b.g = load_vec<T, 4>(static_cast<const T*>(t.g) + at, have);
  if constexpr (MASTER) b.p32 = load_vec<float, 4>(t.master + at, have);
  else b.p16 = load_vec<T, 4>(static_cast<T*>(t.p) + at, have);
  const unsigned char *pm = static_cast<unsigned char*>(t.m) + at, *pv = static_cast<unsigned char*>(t.v) + at;
  if (have == 4) {
    b.cm = *reinterpret_cast<const packed_codes*>(pm);
    b.cv = *reinterpret_cast<const packed_codes*>(pv);
  } else {
    b.cm = b.cv = 0;
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < have) { b.cm |= (uint32_t)pm[e] << (8 * e); b.cv |= (uint32_t)pv[e] << (8 * e); }
  }
  b.sm = t.scale[2 * block];
  b.sv = t.scale[2 * block + 1];
  return b;
}

struct Adamw8Step { double b1, c1, b2, c2; float size, root, decay, eps; uint32_t step; bool careful; };

template <typename T, bool MASTER, bool FULL>
__device__ __forceinline__ void adamw8_block(const AdamwTensor& t, const Adamw8Step& h, const Adamw8Block<T>& now, int64_t block, int64_t i, int have) {
#pragma clang fp contract(off)
  if (FULL) have = 4;
  const double km = (double)now.sm * (1.0 / kTopM), kv = (double)now.sv * (1.0 / kTopV);
  float p[4];
  double m[4], v[4];
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = (int)(now.cm << (24 - 8 * e)) >> 24;
    const uint32_t d = (now.cv >> (8 * e)) & 255u, w = mul_small(d, d);
    const double ge = (double)now.g[e];
    m[e] = h.b1 * ((double)__mul24(c, c < 0 ? -c : c) * km) + h.c1 * ge;
    v[e] = h.b2 * ((double)mul_small(w, w) * kv) + h.c2 * (ge * ge);
    top_m = std::max(top_m, __float_as_uint((float)m[e]) & 0x7FFFFFFFu);
    top_v = std::max(top_v, __float_as_uint((float)v[e]));
    p[e] = adamw_weight(MASTER ? now.p32[e] : now.p16[e], (float)m[e], (float)v[e], h.size, h.root, h.decay, h.eps, h.careful);
  }
  const float sm = adamw_scale(wave_max_bits(top_m)), sv = adamw_scale(wave_max_bits(top_v));
  // both reciprocals by one division: one half of the wave forms each
  const float top = threadIdx.x & 32 ? sv : sm;
  const double inverse = top > 0.f ? 1.0 / (double)top : 0.0;
  const double rm = kTopM * wave_lane(inverse, 0) * 131072.0, rv = kTopV * wave_lane(inverse, 32) * 131072.0;
  uint32_t cm = 0, cv = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t z = adamw_mix((uint32_t)(i + e), h.step);
    const int c = adamw_code_m(fabs(m[e]) * rm, z & 0xFFFFu), d = adamw_code_v(v[e] * rv, z >> 16);
    cm |= ((uint32_t)(m[e] < 0.0 ? -c : c) & 255u) << (8 * e);
    cv |= (uint32_t)(d == 0 && v[e] > 0.0 ? 1 : d) << (8 * e);
  }
  if (have) {
    unsigned char *pm = static_cast<unsigned char*>(t.m) + i, *pv = static_cast<unsigned char*>(t.v) + i;
    if (have == 4) {
      *reinterpret_cast<packed_codes*>(pm) = cm;
      *reinterpret_cast<packed_codes*>(pv) = cv;
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < have) { pm[e] = (unsigned char)(cm >> (8 * e)); pv[e] = (unsigned char)(cv >> (8 * e)); }
    }
    store_vec<T, 4>(static_cast<T*>(t.p) + i, p, have);
    if constexpr (MASTER) store_vec<float, 4>(t.master + i, p, have);
  }
  if ((threadIdx.x & 63) == 0) {
    t.scale[2 * block] = sm;
    t.scale[2 * block + 1] = sv;
  }
}

template <typename T, bool MASTER>
__device__ __forceinline__ void adamw8_chunk(const AdamwArgs& a, const AdamwTensor& t, int k) {
  Adamw8Step h = {a.b1, 1.0 - a.b1, a.b2, 1.0 - a.b2, a.correction[4 * k], a.correction[4 * k + 1], a.decay, a.eps,
                  __float_as_uint(a.correction[4 * k + 2]), adamw_careful(a.eps)};
  asm("" : "+v"(h.eps));      // (in a vector register: an operation takes one scalar)
  // a wave takes a block of 256 elements at a time, four neighbouring ones a lane; the next block's loads are in flight meanwhile
  const int64_t full = t.n / kAdamwBlock, first = (int64_t)(blockIdx.x - a.first[k]) * (kAdamwChunk / kAdamwBlock);
  const int64_t end = std::min<int64_t>(full, first + kAdamwChunk / kAdamwBlock);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t block = first + wave;
  if (block < end) {
    Adamw8Block<T> next = adamw8_load<T, MASTER, true>(t, block, block * kAdamwBlock + lane * 4, 4);
#pragma unroll 1
    for (; block < end; block += 4) {
      const Adamw8Block<T> now = next;
      if (block + 4 < end) next = adamw8_load<T, MASTER, true>(t, block + 4, (block + 4) * kAdamwBlock + lane * 4, 4);
      adamw8_block<T, MASTER, true>(t, h, now, block, block * kAdamwBlock + lane * 4, 4);
    }
  }
  // the tensor's last block, where it is not a whole one
  if (block == full && block < first + kAdamwChunk / kAdamwBlock && full * kAdamwBlock < t.n) {
    const int64_t i = block * kAdamwBlock + lane * 4;
    const int have = (int)std::max<int64_t>(0, std::min<int64_t>(4, t.n - i));
    adamw8_block<T, MASTER, false>(t, h, adamw8_load<T, MASTER, false>(t, block, i, have), block, i, have);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamwArgs a) {
  const int k = adamw_tensor(a.first, a.count, blockIdx.x);
  const AdamwTensor t = a.tensor[k];
  if constexpr (sizeof(T) == 2)
    if (t.master) return adamw8_chunk<T, true>(a, t, k);
  adamw8_chunk<T, false>(a, t, k);
}

// 8-bit states as the values they stand for: 2 bytes in, 8 out an element
__global__ __launch_bounds__(256) void adamw8_values_kernel(const AdamwValuesArgs a) {
  const int k = adamw_tensor(a.first, a.count, blockIdx.x);
  const int64_t n = a.n[k], begin = (int64_t)(blockIdx.x - a.first[k]) * kAdamwChunk + threadIdx.x * 4;
  const unsigned char* cm = static_cast<const unsigned char*>(a.m[k]);
  const unsigned char* cv = static_cast<const unsigned char*>(a.v[k]);
  const float* scale = a.scale[k];
  float *out_m = a.out_m[k], *out_v = a.out_v[k];
  constexpr int R = kAdamwChunk / 1024;
  auto put = [&](int64_t i, uint32_t bm, uint32_t bv, float sm, float sv, int have) {
    const double km = (double)sm * (1.0 / kTopM), kv = (double)sv * (1.0 / kTopV);
    float m[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = (int)(bm << (24 - 8 * e)) >> 24;
      const uint32_t d = (bv >> (8 * e)) & 255u, w = mul_small(d, d);
      m[e] = (float)((double)__mul24(c, c < 0 ? -c : c) * km);
      v[e] = (float)((double)mul_small(w, w) * kv);
    }
    store_vec<float, 4>(out_m + i, m, have);
    store_vec<float, 4>(out_v + i, v, have);
  };
  if ((int64_t)(blockIdx.x - a.first[k] + 1) * kAdamwChunk <= n) {
    uint32_t bm[R], bv[R];
    float sm[R], sv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t i = begin + r * 1024;
      bm[r] = *reinterpret_cast<const packed_codes*>(cm + i);
      bv[r] = *reinterpret_cast<const packed_codes*>(cv + i);
      sm[r] = scale[2 * (i / kAdamwBlock)];
      sv[r] = scale[2 * (i / kAdamwBlock) + 1];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) put(begin + r * 1024, bm[r], bv[r], sm[r], sv[r], 4);
    return;
  }
  for (int64_t i = begin; i < n && i < begin + kAdamwChunk; i += 1024) {
    const int have = (int)std::min<int64_t>(4, n - i);
    uint32_t bm = 0, bv = 0;
    for (int e = 0; e < have; ++e) {
      bm |= (uint32_t)cm[i + e] << (8 * e);
      bv |= (uint32_t)cv[i + e] << (8 * e);
    }
    put(i, bm, bv, scale[2 * (i / kAdamwBlock)], scale[2 * (i / kAdamwBlock) + 1], have);
  }
}

static inline int64_t adamw_chunks(int64_t n) { return (n + kAdamwChunk - 1) / kAdamwChunk; }
// the workgroups of a launch, whose threads are counted in 32 bits (a tensor of them all: 2^36 elements)
constexpr int64_t kAdamwGroups = UINT32_MAX / 256;

}  // namespace socmx

using namespace socmx;

// the counts next to each other (steps), or each of them by its address (counts)
static int adamw_update(int32_t type, int32_t bits, const socmx_adamw_tensor* tensors, int32_t ntensors, float* steps, float* const* counts,
                        float* workspace, double lr, double beta1, double beta2, double eps, double weight_decay, void* stream) {
  if (!tensors || (!steps && !counts) || !workspace) return SOCMX_E_NULL;
  if (type < SOCMX_F32 || type > SOCMX_F16 || (bits != 32 && bits != 8)) return SOCMX_E_KIND;
  if (ntensors < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return SOCMX_E_DIM;
  for (int i = 0; i < ntensors; ++i) {
    const socmx_adamw_tensor& t = tensors[i];
    if (counts && !counts[i]) return SOCMX_E_NULL;
    if (t.n < 0 || t.n > kAdamwGroups * kAdamwChunk) return SOCMX_E_DIM;
    if (t.n == 0) continue;
    if (!t.p || !t.grad || !t.exp_avg || !t.exp_avg_sq || (bits == 8 && !t.scale)) return SOCMX_E_NULL;
    if (t.master && type == SOCMX_F32) return SOCMX_E_KIND;
  }
  // (b = 0: log = -inf, expm1 = -1, the correction is 1)
  const double log_b1 = log(beta1), log_b2 = log(beta2);
  if (steps) {
    if (const int err = launch(adamw_begin_kernel<AdamwSteps>, dim3((ntensors + 63) / 64), dim3(64), 0, stream, AdamwSteps{steps}, (int)ntensors,
                               log_b1, log_b2, lr, workspace))
      return err;
  } else {
    for (int first = 0; first < ntensors; first += kAdamwCounts) {
      const int n = std::min(kAdamwCounts, ntensors - first);
      AdamwCounts some = {};
      std::copy(counts + first, counts + first + n, some.at);
      if (const int err = launch(adamw_begin_kernel<AdamwCounts>, dim3((n + 63) / 64), dim3(64), 0, stream, some, n, log_b1, log_b2, lr,
                                 workspace + 4 * (int64_t)first))
        return err;
    }
  }
  int at = 0;
  while (at < ntensors) {
    AdamwArgs a;
    a.b1 = beta1; a.b2 = beta2; a.decay = (float)(lr * weight_decay); a.eps = (float)eps;
    a.correction = workspace + 4 * (int64_t)at;
    int64_t blocks = 0;
    int count = 0;
    for (; count < kAdamwTensors && at + count < ntensors; ++count) {
      const socmx_adamw_tensor& t = tensors[at + count];
      const int64_t more = adamw_chunks(t.n);
      if (blocks + more > kAdamwGroups) break;
      a.tensor[count] = AdamwTensor{t.p, t.grad, t.exp_avg, t.exp_avg_sq, t.scale, t.master, t.n};
      a.first[count] = (int32_t)blocks;
      blocks += more;
    }
    a.first[count] = (int32_t)blocks;
    a.count = count;
    const dim3 grid((unsigned)blocks), block(256);
    int err = 0;
    if (blocks == 0) {
      // (nothing but empty tensors)
    } else if (type == SOCMX_F32)
      err = bits == 8 ? launch(adamw8_kernel<float>, grid, block, 0, stream, a) : launch(adamw_kernel<float>, grid, block, 0, stream, a);
    else if (type == SOCMX_BF16)
      err = bits == 8 ? launch(adamw8_kernel<bf16_t>, grid, block, 0, stream, a) : launch(adamw_kernel<bf16_t>, grid, block, 0, stream, a);
    else
      err = bits == 8 ? launch(adamw8_kernel<f16_t>, grid, block, 0, stream, a) : launch(adamw_kernel<f16_t>, grid, block, 0, stream, a);
    if (err) return err;
    at += count;
  }
  return 0;
}

extern "C" int socmx_adamw_step(int32_t type, int32_t bits, const socmx_adamw_tensor* tensors, int32_t ntensors, float* steps,
                                float* workspace, double lr, double beta1, double beta2, double eps, double weight_decay,
                                socmx_stream_t stream) {
  return adamw_update(type, bits, tensors, ntensors, steps, nullptr, workspace, lr, beta1, beta2, eps, weight_decay, stream);
}

extern "C" int socmx_adamw_step_counts(int32_t type, int32_t bits, const socmx_adamw_tensor* tensors, int32_t ntensors, float* const* steps,
                                       float* workspace, double lr, double beta1, double beta2, double eps, double weight_decay,
                                       socmx_stream_t stream) {
  return adamw_update(type, bits, tensors, ntensors, nullptr, steps, workspace, lr, beta1, beta2, eps, weight_decay, stream);
}

extern "C" int socmx_adamw_state_values(const socmx_adamw_state* states, int32_t nstates, socmx_stream_t stream) {
  if (!states) return SOCMX_E_NULL;
  if (nstates < 1) return SOCMX_E_DIM;
  for (int i = 0; i < nstates; ++i) {
    const socmx_adamw_state& t = states[i];
    if (t.n < 1 || t.n > kAdamwGroups * kAdamwChunk) return SOCMX_E_DIM;
    if (!t.exp_avg || !t.exp_avg_sq || !t.scale || !t.out_exp_avg || !t.out_exp_avg_sq) return SOCMX_E_NULL;
  }
  int at = 0;
  while (at < nstates) {
    AdamwValuesArgs a;
    int64_t blocks = 0;
    int count = 0;
    for (; count < kAdamwTensors && at + count < nstates; ++count) {
      const socmx_adamw_state& t = states[at + count];
      const int64_t more = adamw_chunks(t.n);
      if (blocks + more > kAdamwGroups) break;
      a.m[count] = t.exp_avg; a.v[count] = t.exp_avg_sq; a.scale[count] = t.scale;
      a.out_m[count] = t.out_exp_avg; a.out_v[count] = t.out_exp_avg_sq; a.n[count] = t.n;
      a.first[count] = (int32_t)blocks;
      blocks += more;
    }
    a.first[count] = (int32_t)blocks;
    a.count = count;
    if (const int err = launch(adamw8_values_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a)) return err;
    at += count;
  }
  return 0;
}
