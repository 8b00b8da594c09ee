// Element types and unaligned vector access shared by the kernels that take fp32, bf16 and fp16
// tensors (layer norm, dropout, rotary positions, attention).
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// 16 bytes of T.  The alignment of one element is enough: rows of odd length and views that
// start anywhere take the same 16-byte global accesses (the hardware splits the ones that cross
// a line), so that layer norm, dropout and rotary positions have one variant for all of them.
// (Attention has two: loads straight to LDS need aligned 16-byte chunks.)
template <typename T>
struct Vec16 {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T utype __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// `cnt` (0..N) elements from p, zeros behind them.
template <typename T>
__device__ __forceinline__ typename Vec16<T>::type load_raw(const T* p, int cnt) {
  if (cnt == Vec16<T>::N) return *reinterpret_cast<const typename Vec16<T>::utype*>(p);
  typename Vec16<T>::type v;
#pragma unroll
  for (int e = 0; e < Vec16<T>::N; ++e) v[e] = e < cnt ? p[e] : (T)0.f;
  return v;
}

// `cnt` (0..N) elements from p as fp32, zeros behind them.
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int cnt, float* out) {
  constexpr int N = Vec16<T>::N;
  if (cnt == N) {
    const typename Vec16<T>::utype v = *reinterpret_cast<const typename Vec16<T>::utype*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = e < cnt ? (float)p[e] : 0.f;
  }
}

// The first `cnt` (0..N) of N fp32 values to p, rounded once to nearest even.
template <typename T>
__device__ __forceinline__ void store_vec(T* p, int cnt, const float* in) {
  constexpr int N = Vec16<T>::N;
  if (cnt == N) {
    typename Vec16<T>::utype v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (T)in[e];
    *reinterpret_cast<typename Vec16<T>::utype*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < cnt) p[e] = (T)in[e];
  }
}

// v of lane l plus v of lane l ^ 32 (or l ^ 16), without LDS.
__device__ __forceinline__ float plus_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float plus_xor16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over groups of LANES (8 .. 64) neighbouring lanes, in every lane of the group: within 16
// lanes by DPP (neighbour, pair, mirrored half row, mirrored row), across them by lane swaps - a
// few cycles each where a shuffle through LDS takes a hundred.  A group reads its own lanes only.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  v = plus_dpp<0xB1>(v);
  v = plus_dpp<0x4E>(v);
  v = plus_dpp<0x141>(v);
  if (LANES > 8) v = plus_dpp<0x140>(v);
  if (LANES > 16) v = plus_xor16(v);
  if (LANES > 32) v = plus_xor32(v);
  return v;
}

// The same for 64 bits and a whole wave: each half of a number moves like a float.
__device__ __forceinline__ double from_halves(uint32_t lo, uint32_t hi) {
  return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}
template <int CTRL>
__device__ __forceinline__ double plus_dpp(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, true);
  return v + from_halves((uint32_t)lo, (uint32_t)hi);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = plus_dpp<0xB1>(v);
  v = plus_dpp<0x4E>(v);
  v = plus_dpp<0x141>(v);
  v = plus_dpp<0x140>(v);
  uint64_t b = (uint64_t)__double_as_longlong(v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  v = from_halves(lo[0], hi[0]) + from_halves(lo[1], hi[1]);
  b = (uint64_t)__double_as_longlong(v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  return from_halves(lo[0], hi[0]) + from_halves(lo[1], hi[1]);
}

// Calls f with a value of the element type that `dtype` names; MN_EUNSUPPORTED for others.
template <typename F>
static inline int mn_for_dtype(int dtype, F f) {
  switch (dtype) {
    case MN_F32: return f(float());
    case MN_BF16: return f(bf16_t());
    case MN_F16: return f(f16_t());
    default: return MN_EUNSUPPORTED;
  }
}
