// Dropout from a counter-based generator: whether an element stays is a function of (seed,
// offset, element number), so the backward pass and a recomputed forward ask the generator again
// and no mask is ever stored.
//
//   u(e) = 32-bit number of element e;  keep(e) = u(e) >= round(p * 2^32);  y = keep ? x / (1-p) : 0
//
// u comes from Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1,
// 2, 3", SC 2011).  Eight elements share a counter (e / 8, offset) under the key `seed`: its four
// words give each element the HIGH half of its number, and the low halves - the same counter with
// bit 31 of its second word set - are only generated where a high half equals the threshold's,
// one element in 65536, since anywhere else the high half decides.  A word per element instead
// would cost twice the multiplications, more time than the memory of 16-bit tensors takes.
// Bound by memory: one read and one write per element, 16 bytes a lane and load: 36064 x 4096 bf16
// in 102 us (5.8 TB/s; a copy of 1 GiB runs at 5.0), 10868 x 1023 fp32 in 15 us a direction.
#include "elem.h"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4_t philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                                 uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return uint4_t{c0, c1, c2, c3};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const T* x, T* y, int64_t n,
                                                           const uint64_t* __restrict__ state,
                                                           uint32_t threshold, float scale) {
  constexpr int N = Vec16<T>::N;
  const uint64_t seed = state[0], offset = state[1];
  const uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  const uint32_t o0 = (uint32_t)offset, o1 = (uint32_t)(offset >> 32);
  const uint32_t high = threshold >> 16, low = threshold & 0xFFFFu;
  const int64_t groups = (n + 7) / 8;
  for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < groups;
       g += (int64_t)gridDim.x * kThreads) {
    const int64_t e0 = g * 8;
    const int cnt = n - e0 >= 8 ? 8 : (int)(n - e0);
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; c += N) {
      const int k = cnt - c;
      load_vec<T>(x + e0 + c, k >= N ? N : (k > 0 ? k : 0), v + c);
    }
    const uint4_t w = philox4x32_10((uint32_t)g, (uint32_t)(g >> 32), o0, o1, k0, k1);
    uint32_t h[8];
    bool tie = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
      tie |= h[e] == high;
    }
    uint32_t keep = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) keep |= (h[e] > high ? 1u : 0u) << e;
    if (tie) {
      const uint4_t l = philox4x32_10((uint32_t)g, (uint32_t)(g >> 32) | 0x80000000u, o0, o1, k0, k1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t le = e & 1 ? l[e / 2] >> 16 : l[e / 2] & 0xFFFFu;
        if (h[e] == high && le >= low) keep |= 1u << e;
      }
    }
    // (a choice, not a product: a dropped infinity or NaN is zero)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = keep >> e & 1 ? v[e] * scale : 0.f;
#pragma unroll
    for (int c = 0; c < 8; c += N) {
      const int k = cnt - c;
      store_vec<T>(y + e0 + c, k >= N ? N : (k > 0 ? k : 0), v + c);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void zero_all_kernel(T* y, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kThreads)
    y[i] = (T)0.f;
}

}  // namespace

extern "C" {

int mn_dropout(const void* x, void* y, int64_t n, double p, const uint64_t* state, int dtype,
               mn_stream_t stream) {
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return MN_EINVAL;
  if (n >= (1ll << 60)) return MN_EUNSUPPORTED;
  return mn_for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (n == 0) return (int)MN_OK;
    if (!x || !y || !state) return (int)MN_EINVAL;
    hipStream_t s = mn_stream(stream);
    const int64_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
    const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
    const double scaled = p * 4294967296.0 + 0.5;
    if (scaled >= 4294967296.0) {   // no number reaches the threshold: nothing stays (p = 1 among them)
      zero_all_kernel<T><<<grid, kThreads, 0, s>>>((T*)y, n);
      return mn_launch_status();
    }
    const uint32_t threshold = (uint32_t)scaled;
    dropout_kernel<T><<<grid, kThreads, 0, s>>>((const T*)x, (T*)y, n, state, threshold,
                                                (float)(1.0 / (1.0 - p)));
    return mn_launch_status();
  });
}

}  // extern "C"
