// Rotary positions over several axes (row and column of an image's patches, frame of a video).
//
// The first 2*n elements of a head are n pairs, (i, i+n) or, interleaved, (2i, 2i+1); pair i is
// turned by the angle position[axis(i)] * frequency(i), the rest is copied.  Backward turns the
// other way, so it is the same kernel with the sign of the sine changed.
//
// Bound by memory: one read, one write.  What could cost more are the angles: they are needed
// once per (token, pair) but used by every head and, where positions do not depend on the batch,
// by every batch entry, so a workgroup makes a table of cosines and sines for TOK tokens in LDS
// and walks over heads and entries of the batch with it.
// Angles are held in TURNS in 64 bits: position * (frequency / 2 pi) leaves its whole turns and
// quarter turns exactly (what is left is at most an eighth of a turn, 2^-28 turns after rounding
// to fp32), so a position of a million is as accurate as position 1; sine and cosine of that rest
// are fp32.
// 184 x 196 tokens of 16 heads of 64, bf16: 34 us on operands from memory (4.3 TB/s), 27 us on ones
// in the memory-side cache; 6916 tokens of 12 heads of 80, fp32: 14 us (3.8 TB/s; one round of
// workgroups, half of it the wait for the table and the first loads).  With what a unit is worked
// out for every element instead of once per lane the latter took 20 us.
#include <math.h>

#include "elem.h"

namespace {

constexpr int kThreads = 256;
constexpr int kSlots = 4;
constexpr int kBlockElems = 4096;
constexpr int kMaxPairs = 128;
constexpr int64_t kMaxToken = 1 << 24;   // elements of a token
constexpr int kTableFloats = 8192;   // 32 KB of LDS: TOK * pairs * 2

struct Rotary {
  double turns[kMaxPairs];    // frequency / (2 pi)
  uint8_t axis[kMaxPairs];
  int64_t B, T;
  int64_t sxb, sxt, sxh;      // strides of x in elements
  int64_t spa, spb, spt;      // strides of the positions
  int32_t H, D, n, tok, bchunk;
  float sign;
};

template <typename P>
__device__ __forceinline__ float2_t cos_sin(P pos, double turns) {
  double t = (double)pos * turns;
  t -= rint(t);                                  // [-1/2, 1/2]
  const double quarter = rint(4.0 * t);          // -2 .. 2
  const float rest = (float)(t - 0.25 * quarter) * 2.f;   // half turns, |rest| <= 1/4
  float s, c;
  sincospif(rest, &s, &c);
  switch ((int)quarter & 3) {
    case 0: return float2_t{c, s};
    case 1: return float2_t{-s, c};
    case 2: return float2_t{-c, -s};
    default: return float2_t{s, -c};
  }
}

template <typename T, typename P, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                          const P* __restrict__ pos, const Rotary a) {
  constexpr int N = Vec16<T>::N;
  extern __shared__ float2_t table[];   // [tok][n]
  const int64_t t0 = (int64_t)blockIdx.x * a.tok, b0 = (int64_t)blockIdx.y * a.bchunk;
  const int toks = a.T - t0 < a.tok ? (int)(a.T - t0) : a.tok;
  const int batches = a.B - b0 < a.bchunk ? (int)(a.B - b0) : a.bchunk;
  for (int i = threadIdx.x; i < toks * a.n; i += kThreads) {
    const int t = i / a.n, k = i - t * a.n;
    float2_t cs = cos_sin<P>(pos[a.axis[k] * a.spa + b0 * a.spb + (t0 + t) * a.spt], a.turns[k]);
    cs[1] *= a.sign;
    table[i] = cs;
  }
  __syncthreads();
  // Units of a head: chunks of N pairs, then chunks that are copied; interleaved, chunks of N
  // elements, where what is copied is a pair that turns by nothing (so that only the end of a head
  // is less than 16 bytes).
  // A wave takes a token at a time, a lane the same kSlots units of each, so that what a unit is
  // and where it lies is worked out once; tokens of at most 64 units are taken kSlots at a time.
  // All loads of a turn are on their way before the first is used.
  const int pair_units = INTERLEAVED ? (a.D + N - 1) / N : (a.n + N - 1) / N;
  const int units = INTERLEAVED ? pair_units : pair_units + (a.D - 2 * a.n + N - 1) / N, per_token = a.H * units;
  const int wave = threadIdx.x / MN_WAVE, lane = threadIdx.x % MN_WAVE, waves = kThreads / MN_WAVE;
  const bool narrow = per_token <= MN_WAVE;
  const int tokens = batches * toks, step = narrow ? waves * kSlots : waves;
  for (int first = 0; first < per_token; first += narrow ? MN_WAVE : MN_WAVE * kSlots) {
    int64_t xo[kSlots];
    int yo[kSlots], tab[kSlots], cnt[kSlots];   // cnt: elements (of either half of the pairs); 0: nothing
    bool copy[kSlots];
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
      const int hu = first + (narrow ? 0 : k * MN_WAVE) + lane;
      const int h = hu / units, u = hu - h * units;
      copy[k] = !INTERLEAVED && u >= pair_units;
      const int col = copy[k] ? 2 * a.n + (u - pair_units) * N : u * N;
      xo[k] = h * a.sxh + col;
      yo[k] = h * a.D + col;
      tab[k] = INTERLEAVED ? col / 2 : col;   // first pair
      const int left = (INTERLEAVED || copy[k] ? a.D : a.n) - col;
      cnt[k] = hu < per_token ? (left < N ? left : N) : 0;
    }
    for (int bt0 = wave; bt0 < tokens; bt0 += step) {
      typename Vec16<T>::type lo[kSlots], hi[kSlots];
#pragma unroll
      for (int k = 0; k < kSlots; ++k) {
        const int bt = bt0 + (narrow ? k * waves : 0);
        if (bt >= tokens || cnt[k] == 0) continue;
        const int bi = bt / toks, t = bt - bi * toks;
        const T* p = x + (b0 + bi) * a.sxb + (t0 + t) * a.sxt + xo[k];
        lo[k] = load_raw<T>(p, cnt[k]);
        if (!INTERLEAVED && !copy[k]) hi[k] = load_raw<T>(p + a.n, cnt[k]);
      }
#pragma unroll
      for (int k = 0; k < kSlots; ++k) {
        const int bt = bt0 + (narrow ? k * waves : 0);
        if (bt >= tokens || cnt[k] == 0) continue;
        const int bi = bt / toks, t = bt - bi * toks;
        T* q = y + ((b0 + bi) * a.T + t0 + t) * (int64_t)(a.H * a.D) + yo[k];
        float v[N];
        if (copy[k]) {
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = (float)lo[k][e];
          store_vec<T>(q, cnt[k], v);
          continue;
        }
        const float2_t* cs = table + t * a.n + tab[k];
        if (INTERLEAVED) {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) {
            const bool turns = tab[k] + e < a.n;
            const float2_t c = turns ? cs[e] : float2_t{1.f, 0.f};
            const float f = (float)lo[k][2 * e], g = (float)lo[k][2 * e + 1];
            v[2 * e] = turns ? f * c[0] - g * c[1] : f;   // (a copied infinity is no pair's)
            v[2 * e + 1] = turns ? f * c[1] + g * c[0] : g;
          }
          store_vec<T>(q, cnt[k], v);
        } else {
          float w[N];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float2_t c = cs[e < cnt[k] ? e : 0];
            const float f = (float)lo[k][e], g = (float)hi[k][e];
            v[e] = f * c[0] - g * c[1];
            w[e] = f * c[1] + g * c[0];
          }
          store_vec<T>(q, cnt[k], v);
          store_vec<T>(q + a.n, cnt[k], w);
        }
      }
    }
  }
}

}  // namespace

extern "C" {

int mn_rotary(const mn_rotary_desc* d, const void* x, const void* positions, void* y, int inverse,
              int dtype, mn_stream_t stream) {
  if (!d) return MN_EINVAL;
  if (d->B < 0 || d->T < 0 || d->H < 0 || d->D <= 0 || d->axes < 1 || d->axes > 3 || !(d->base > 0.0))
    return MN_EINVAL;
  int64_t n = 0;
  for (int k = 0; k < d->axes; ++k) {
    if (d->sections[k] < 0) return MN_EINVAL;
    n += d->sections[k];
  }
  if (2 * n > d->D) return MN_EINVAL;
  if (n > kMaxPairs || (int64_t)d->H * d->D >= kMaxToken || d->B >= (1ll << 31) || d->T >= (1ll << 31))
    return MN_EUNSUPPORTED;
  if (d->pos_type < MN_POS_I64 || d->pos_type > MN_POS_F32) return MN_EUNSUPPORTED;
  Rotary a = {};
  int k = 0;
  for (int axis = 0; axis < d->axes; ++axis)
    for (int i = 0; i < d->sections[axis]; ++i, ++k) {
      const double power = d->joint ? (double)k / (double)n : (double)i / (double)d->sections[axis];
      a.turns[k] = pow(d->base, -power) * 0.15915494309189533577;   // 1 / (2 pi)
      a.axis[k] = (uint8_t)axis;
    }
  a.B = d->B; a.T = d->T; a.H = d->H; a.D = d->D; a.n = (int)n;
  a.sxb = d->x_stride[0]; a.sxt = d->x_stride[1]; a.sxh = d->x_stride[2];
  a.spa = d->pos_stride[0]; a.spb = d->pos_stride[1]; a.spt = d->pos_stride[2];
  a.sign = inverse ? -1.f : 1.f;
  // tokens of a workgroup: about kBlockElems elements of x, as far as the table has room; entries of the
  // batch share the table unless their positions differ, as long as 2048 workgroups remain
  const int64_t token_elems = (int64_t)a.H * a.D;
  int64_t tok = token_elems ? kBlockElems / token_elems : 1;
  const int64_t room = n ? kTableFloats / (2 * n) : 64;
  tok = tok < 1 ? 1 : (tok > room ? room : (tok > 64 ? 64 : tok));
  if (tok > a.T) tok = a.T > 0 ? a.T : 1;
  a.tok = (int)tok;
  const int64_t tblocks = (a.T + tok - 1) / tok;
  int64_t bchunk = 1;
  if (a.spb == 0) {
    bchunk = a.B * tblocks / 2048;
    bchunk = bchunk < 1 ? 1 : bchunk;
  }
  // (the grid's second dimension ends at 65535, a workgroup's elements are counted in 32 bits)
  while ((a.B + bchunk - 1) / bchunk > 65535 && a.spb == 0) bchunk *= 2;
  const int64_t most = token_elems ? (1ll << 31) / (tok * token_elems) - 1 : bchunk;
  if (bchunk > most) bchunk = most;
  // (threads of a launch are counted in 32 bits)
  if ((a.B + bchunk - 1) / bchunk > 65535 || tblocks > ((1ll << 32) - 1) / kThreads) return MN_EUNSUPPORTED;
  a.bchunk = (int)(bchunk < a.B ? bchunk : a.B);
  return mn_for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.B == 0 || a.T == 0 || a.H == 0) return (int)MN_OK;
    if (!x || !positions || !y) return (int)MN_EINVAL;
    const dim3 grid((unsigned)tblocks, (unsigned)((a.B + a.bchunk - 1) / a.bchunk));
    const size_t lds = (size_t)a.tok * a.n * sizeof(float2_t);
    hipStream_t s = mn_stream(stream);
    const auto launch = [&](auto p) {
      using P = decltype(p);
      if (d->interleaved)
        rotary_kernel<T, P, true><<<grid, kThreads, lds, s>>>((const T*)x, (T*)y, (const P*)positions, a);
      else
        rotary_kernel<T, P, false><<<grid, kThreads, lds, s>>>((const T*)x, (T*)y, (const P*)positions, a);
      return mn_launch_status();
    };
    if (d->pos_type == MN_POS_I64) return launch(int64_t());
    if (d->pos_type == MN_POS_I32) return launch(int32_t());
    return launch(float());
  });
}

}  // extern "C"
