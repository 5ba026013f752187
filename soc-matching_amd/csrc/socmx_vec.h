// socmx_vec.h -- element types of the layer operators (f32, bf16, f16), vectors of them in memory, sums over groups of lanes.
//
// A vector access needs the alignment of ONE element only: gfx950 loads and stores 4, 8 and 16 bytes at any address, an
// access that crosses a cache line costs a second one.  Rows at odd offsets (slices, tensors packed in flat buffers)
// therefore take the same kernels as aligned ones.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace socmx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int N>
struct mem_vec {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T>
struct mem_vec<T, 1> { typedef T type; };

template <typename T, int N>
struct reg_vec {                                    // N elements as they stand in memory
  typename mem_vec<T, N>::type v;
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (N == 1) return (float)v; else return (float)v[i];
  }
};

template <typename T, int N>
__device__ __forceinline__ reg_vec<T, N> load_vec(const T* p) {
  reg_vec<T, N> r;
  r.v = *reinterpret_cast<const typename mem_vec<T, N>::type*>(p);
  return r;
}

// the first `n` of N elements, zeros behind them
template <typename T, int N>
__device__ __forceinline__ reg_vec<T, N> load_vec(const T* p, int n) {
  if (n >= N) return load_vec<T, N>(p);
  reg_vec<T, N> r;
  if constexpr (N == 1) {
    r.v = (T)0.f;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

// rounds to T (to nearest, ties to even)
template <typename T, int N>
__device__ __forceinline__ typename mem_vec<T, N>::type round_vec(const float (&x)[N]) {
  typename mem_vec<T, N>::type v;
  if constexpr (N == 1) {
    v = (T)x[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
  }
  return v;
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  *reinterpret_cast<typename mem_vec<T, N>::type*>(p) = round_vec<T, N>(x);
}

// for what the kernel writes once and nothing near reads: it takes no cache lines from the loads
template <typename T, int N>
__device__ __forceinline__ void stream_vec(T* p, const float (&x)[N]) {
  __builtin_nontemporal_store(round_vec<T, N>(x), reinterpret_cast<typename mem_vec<T, N>::type*>(p));
}

template <typename T, int N>
__device__ __forceinline__ void stream_vec(T* p, const float (&x)[N], int n) {
  if (n >= N) {
    stream_vec<T, N>(p, x);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (T)x[i];
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N], int n) {
  if (n >= N) {
    store_vec<T, N>(p, x);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (T)x[i];
}

// ---- sums over 8, 16, 32 or 64 neighbouring lanes; every lane of the group ends with the total -----------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(L == 1 || L == 2 || L == 4 || L == 8 || L == 16 || L == 32 || L == 64, "a power of two within a wave");
  if constexpr (L >= 2) v += dpp_move<0xB1>(v);      // quad_perm [1,0,3,2]
  if constexpr (L >= 4) v += dpp_move<0x4E>(v);      // quad_perm [2,3,0,1]
  if constexpr (L >= 8) v += dpp_move<0x141>(v);     // mirror of 8 lanes
  if constexpr (L >= 16) v += dpp_move<0x140>(v);    // mirror of 16 lanes
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (L >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

}  // namespace socmx
