// Layer normalisation over the last D elements of every row, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) * r, y = xh * w + b
//   dx = r * (g*w - mean(g*w) - xh * mean(g*w * xh)),  dw = sum_rows g * xh,  db = sum_rows g
//
// Both passes are bound by memory: a row is read once, kept in registers (NE values per lane),
// and written once.  The variance is taken around the mean in a second pass over the registers,
// so a row far off zero loses nothing.  LANES lanes share a row: part of a wave for short rows
// (several rows a wave), a wave up to 2048 elements forward and 1024 backward, a workgroup above, of
// up to 1024 lanes and 16384 elements; the groups walk over the rows with w and b in registers, so those are read once per group and not once per row (with
// fp32 weights next to 16-bit rows they are twice the bytes of the row), and load the next row
// before they work on one.  Longer rows are read again for each sum, an element a lane at a time.
// Backward sums dw and db over a group's rows in registers, over a workgroup's groups in a fixed
// order, and writes one partial row per workgroup; a second kernel adds those in a fixed order:
// no atomics, the same bits every run.  Sums are fp32, of rows too long for registers 64 bits.
// y may lie where x does and dx where g does: those pointers are not declared free of aliases.
//
// 36064 rows x 2048, bf16 with fp32 weights: forward 68 us (4.4 TB/s), backward 92 us (4.8 TB/s)
// and 5 us for the join; 36248 x 384, fp32: 22 us, 29 us (5.1 and 5.8 TB/s) and 4 us; a copy of
// 1 GiB runs at 5.1 TB/s.  Without the next row's loads ahead, and with the sums through LDS, the
// first took 107 and 145 us.
// Wider rows are further from the copy.  Backward with 1024 lanes (8193 .. 16384 elements) has 128
// registers a lane, does not fit and spills 83 to 117 of them to scratch memory.  bf16 with fp32
// weights, forward / backward: 6000 x 8192 in 52 / 109 us (3.8 / 2.7 TB/s), 4096 x 12288 in 86 / 287
// (2.4 / 1.1), 3000 x 16384 in 86 / 291 (2.3 / 1.0); in several passes over a row, 2000 x 16392 in
// 62 / 103 (2.1 / 1.9) and 512 x 150528 in 163 / 359 (1.9 / 1.3).
#include "elem.h"

namespace {

constexpr int kMaxParts = 1024;    // partial rows of dw / db at most
constexpr int kMaxBlocks = 1024;   // forward: four workgroups a CU

// Sum over the LANES lanes (or threads) of a group; every lane gets the total.
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float* lds) {
  v = lane_sum<(LANES < MN_WAVE ? LANES : MN_WAVE)>(v);
  if (LANES > MN_WAVE) {
    __syncthreads();   // the previous sum has been read
    if (threadIdx.x % MN_WAVE == 0) lds[threadIdx.x / MN_WAVE] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / MN_WAVE; ++w) v += lds[w];
  }
  return v;
}

// Two sums at once: one wait for both.
template <int LANES>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* lds) {
  a = lane_sum<(LANES < MN_WAVE ? LANES : MN_WAVE)>(a);
  b = lane_sum<(LANES < MN_WAVE ? LANES : MN_WAVE)>(b);
  if (LANES > MN_WAVE) {
    __syncthreads();
    if (threadIdx.x % MN_WAVE == 0) {
      lds[2 * (threadIdx.x / MN_WAVE)] = a;
      lds[2 * (threadIdx.x / MN_WAVE) + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / MN_WAVE; ++w) {
      a += lds[2 * w];
      b += lds[2 * w + 1];
    }
  }
}

// Where element (chunk c, e) of a lane lies in the row, and how many of the chunk's are in it.
template <int LANES, int N>
__device__ __forceinline__ int chunk_col(int lane, int c) {
  return (c * LANES + lane) * N;
}
template <int N>
__device__ __forceinline__ int chunk_cnt(int64_t D, int col) {
  const int64_t left = D - col;
  return left >= N ? N : (left > 0 ? (int)left : 0);
}

// A lane's part of a row, as it lies in memory.
template <typename T, int LANES, int NE>
struct RowPart {
  static constexpr int N = Vec16<T>::N;
  typename Vec16<T>::type v[NE / N];
  __device__ __forceinline__ void load(const T* row, int64_t D, int lane) {
#pragma unroll
    for (int c = 0; c < NE / N; ++c) {
      const int col = chunk_col<LANES, N>(lane, c);
      v[c] = load_raw<T>(row + col, chunk_cnt<N>(D, col));   // zeros behind the row
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return (float)v[e / N][e % N]; }
};

// NE weights of a lane as fp32 (`none` where there is no weight tensor).
template <typename W, int LANES, int NE, int N>
__device__ __forceinline__ void load_weights(const W* w, int64_t D, int lane, float none, float* out) {
#pragma unroll
  for (int c = 0; c < NE / N; ++c) {
    const int col = chunk_col<LANES, N>(lane, c), cnt = chunk_cnt<N>(D, col);
#pragma unroll
    for (int e = 0; e < N; ++e)
      out[c * N + e] = w ? (e < cnt ? (float)w[col + e] : 0.f) : none;
  }
}

template <typename T, typename W, int LANES, int NE>
__global__ __launch_bounds__(LANES > 64 ? LANES : 256) void ln_fwd_kernel(
    const T* x, const W* __restrict__ w, const W* __restrict__ b, T* y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, int64_t rows, int64_t D, float dim, float eps) {
  constexpr int N = Vec16<T>::N, TPB = LANES > 64 ? LANES : 256, G = TPB / LANES;
  __shared__ float lds[2 * TPB / MN_WAVE];
  const int lane = threadIdx.x % LANES;
  float wr[NE], br[NE];
  load_weights<W, LANES, NE, N>(w, D, lane, 1.f, wr);
  load_weights<W, LANES, NE, N>(b, D, lane, 0.f, br);
  // (the next row is on its way while this one is worked on)
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / LANES;
  RowPart<T, LANES, NE> ahead;
  if (row < rows) ahead.load(x + row * D, D, lane);
  for (; row < rows; row += step) {
    float v[NE];
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      v[e] = ahead[e];
      s += v[e];
    }
    if (row + step < rows) ahead.load(x + (row + step) * D, D, lane);
    const float mu = group_sum<LANES>(s, lds) / dim;
    s = 0.f;
#pragma unroll
    for (int c = 0; c < NE / N; ++c) {
      const int cnt = chunk_cnt<N>(D, chunk_col<LANES, N>(lane, c));
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = v[c * N + e] - mu;
        v[c * N + e] = d;
        s += e < cnt ? d * d : 0.f;
      }
    }
    const float r = 1.f / sqrtf(group_sum<LANES>(s, lds) / dim + eps);
    T* yr = y + row * D;
#pragma unroll
    for (int c = 0; c < NE / N; ++c) {
      const int col = chunk_col<LANES, N>(lane, c);
#pragma unroll
      for (int e = 0; e < N; ++e) v[c * N + e] = v[c * N + e] * r * wr[c * N + e] + br[c * N + e];
      store_vec<T>(yr + col, chunk_cnt<N>(D, col), v + c * N);
    }
    if (lane == 0) {
      if (mean_out) mean_out[row] = mu;
      if (rstd_out) rstd_out[row] = r;
    }
  }
}

// parts == nullptr: the only workgroup, which writes dw / db itself.
template <typename T, typename W, int LANES, int NE>
__global__ __launch_bounds__(LANES > 64 ? LANES : 256) void ln_bwd_kernel(
    const T* g, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const W* __restrict__ w, T* dx,
    float* __restrict__ parts, W* __restrict__ dw, W* __restrict__ db, int64_t rows, int64_t D,
    float dim) {
  constexpr int N = Vec16<T>::N, TPB = LANES > 64 ? LANES : 256, G = TPB / LANES;
  __shared__ float lds[2 * TPB / MN_WAVE];
  const int lane = threadIdx.x % LANES;
  float wr[NE], aw[NE], ab[NE];
  load_weights<W, LANES, NE, N>(w, D, lane, 1.f, wr);
#pragma unroll
  for (int e = 0; e < NE; ++e) aw[e] = ab[e] = 0.f;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / LANES;
  RowPart<T, LANES, NE> xa, ga;   // the next row; zeros behind it add nothing below
  float mu_a = 0.f, r_a = 0.f;
  if (row < rows) {
    xa.load(x + row * D, D, lane);
    ga.load(g + row * D, D, lane);
    mu_a = mean[row];
    r_a = rstd[row];
  }
  for (; row < rows; row += step) {
    const float mu = mu_a, r = r_a;
    float xv[NE], gv[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      xv[e] = xa[e];
      gv[e] = ga[e];
    }
    if (row + step < rows) {
      xa.load(x + (row + step) * D, D, lane);
      ga.load(g + (row + step) * D, D, lane);
      mu_a = mean[row + step];
      r_a = rstd[row + step];
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const float xh = (xv[e] - mu) * r, gg = gv[e];
      xv[e] = xh;
      aw[e] += gg * xh;
      ab[e] += gg;
      gv[e] = gg * wr[e];
      s1 += gv[e];
      s2 += gv[e] * xh;
    }
    group_sum2<LANES>(s1, s2, lds);
    s1 /= dim;
    s2 /= dim;
    if (dx) {
      T* dr = dx + row * D;
#pragma unroll
      for (int c = 0; c < NE / N; ++c) {
        const int col = chunk_col<LANES, N>(lane, c);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int k = c * N + e;
          gv[k] = r * (gv[k] - s1 - xv[k] * s2);
        }
        store_vec<T>(dr + col, chunk_cnt<N>(D, col), gv + c * N);
      }
    }
  }
  if (!parts && !dw && !db) return;
  // the groups of a wave, then the waves one after the other
  if (LANES < MN_WAVE) {
#pragma unroll
    for (int o = MN_WAVE / 2; o >= LANES; o >>= 1)
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        aw[e] += __shfl_xor(aw[e], o, MN_WAVE);
        ab[e] += __shfl_xor(ab[e], o, MN_WAVE);
      }
  }
  constexpr int kWaveGroups = LANES <= MN_WAVE ? TPB / MN_WAVE : 1;   // waves with sums of their own
  if (kWaveGroups > 1) {
    // (a row of at most NE * min(LANES, 64) elements; the last wave ends with the total)
    constexpr int ROW = NE * (LANES < MN_WAVE ? LANES : MN_WAVE);
    __shared__ float acc[kWaveGroups > 1 ? 2 * ROW : 1];
    const int wave = threadIdx.x / MN_WAVE;
    const bool mine = threadIdx.x % MN_WAVE < LANES;
    for (int k = 0; k < kWaveGroups; ++k) {
      __syncthreads();
      if (wave == k && mine) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int i = e * (LANES < MN_WAVE ? LANES : MN_WAVE) + lane;
          if (k > 0) {
            aw[e] += acc[i];
            ab[e] += acc[ROW + i];
          }
          acc[i] = aw[e];
          acc[ROW + i] = ab[e];
        }
      }
    }
    if (wave != kWaveGroups - 1 || !mine) return;
  }
#pragma unroll
  for (int c = 0; c < NE / N; ++c) {
    const int col = chunk_col<LANES, N>(lane, c), cnt = chunk_cnt<N>(D, col);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (e >= cnt) continue;
      if (parts) {
        parts[((int64_t)blockIdx.x * 2) * D + col + e] = aw[c * N + e];
        parts[((int64_t)blockIdx.x * 2 + 1) * D + col + e] = ab[c * N + e];
      } else {
        if (dw) dw[col + e] = (W)aw[c * N + e];
        if (db) db[col + e] = (W)ab[c * N + e];
      }
    }
  }
}

// dw / db = the partial rows added up: 32 columns a workgroup, 32 slices of the partial rows,
// joined in order.  blockIdx.y: 0 = dw, 1 = db.  (A launch counts its threads in 32 bits: the
// workgroups of a very long row walk over the columns.)
constexpr int64_t kJoinBlocks = 1 << 20;
template <typename W>
__global__ __launch_bounds__(1024) void ln_join_kernel(const float* __restrict__ parts, W* dw, W* db,
                                                       int nparts, int64_t D) {
  __shared__ float lds[32][33];
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = threadIdx.x % 32, slice = threadIdx.x / 32;
  for (int64_t col0 = (int64_t)blockIdx.x * 32; col0 < D; col0 += (int64_t)gridDim.x * 32) {
    const int64_t col = col0 + c;
    float s = 0.f;
    if (col < D) {
#pragma unroll 8
      for (int p = slice; p < nparts; p += 32) s += parts[((int64_t)p * 2 + blockIdx.y) * D + col];
    }
    __syncthreads();   // the columns before have been read
    lds[slice][c] = s;
    __syncthreads();
    // the slices of column `slice`, one a lane
    s = lane_sum<32>(lds[c][slice]);
    const int64_t mine = col0 + slice;
    if (c == 0 && mine < D) out[mine] = (W)s;
  }
}

// ------------------------------------------------ rows too long for a workgroup's registers
// A thread adds D / 1024 terms here, and rows / 64 for dw and db: in 64 bits, since a chain of fp32
// additions drifts by up to half a step of its sum with each.
constexpr int kLongThreads = 1024;
constexpr int64_t kLongRows = ((1ll << 32) - 1) / kLongThreads;   // threads of a launch: 32 bits

// Sum over a workgroup; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum64(v);
  __syncthreads();   // the previous sum has been read
  if (threadIdx.x % MN_WAVE == 0) lds[threadIdx.x / MN_WAVE] = v;
  __syncthreads();
  v = 0.;
#pragma unroll
  for (int w = 0; w < kLongThreads / MN_WAVE; ++w) v += lds[w];
  return v;
}

template <typename T, typename W>
__global__ __launch_bounds__(kLongThreads) void ln_fwd_long_kernel(
    const T* x, const W* __restrict__ w, const W* __restrict__ b, T* y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, int64_t D, double dim, float eps) {
  __shared__ double lds[kLongThreads / MN_WAVE];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * D;
  T* yr = y + row * D;
  double s = 0.;
  for (int64_t i = threadIdx.x; i < D; i += kLongThreads) s += (double)(float)xr[i];
  const float mu = (float)(block_sum(s, lds) / dim);
  s = 0.;
  for (int64_t i = threadIdx.x; i < D; i += kLongThreads) {
    const double d = (float)xr[i] - mu;
    s += d * d;
  }
  const float r = 1.f / sqrtf((float)(block_sum(s, lds) / dim) + eps);
  for (int64_t i = threadIdx.x; i < D; i += kLongThreads)
    yr[i] = (T)(((float)xr[i] - mu) * r * (w ? (float)w[i] : 1.f) + (b ? (float)b[i] : 0.f));
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[row] = mu;
    if (rstd_out) rstd_out[row] = r;
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kLongThreads) void ln_bwd_long_kernel(
    const T* g, const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
    const W* __restrict__ w, T* dx, int64_t D, double dim) {
  __shared__ double lds[kLongThreads / MN_WAVE];
  const int64_t row = blockIdx.x;
  const float mu = mean[row], r = rstd[row];
  double a1 = 0., a2 = 0.;
  for (int64_t i = threadIdx.x; i < D; i += kLongThreads) {
    const float gw = (float)g[row * D + i] * (w ? (float)w[i] : 1.f);
    a1 += (double)gw;
    a2 += (double)gw * (double)(((float)x[row * D + i] - mu) * r);
  }
  const float s1 = (float)(block_sum(a1, lds) / dim), s2 = (float)(block_sum(a2, lds) / dim);
  for (int64_t i = threadIdx.x; i < D; i += kLongThreads) {
    const float gw = (float)g[row * D + i] * (w ? (float)w[i] : 1.f);
    dx[row * D + i] = (T)(r * (gw - s1 - ((float)x[row * D + i] - mu) * r * s2));
  }
}

// Partial sums of dw / db for one slice of the rows (blockIdx.y), one thread per column.
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_kernel(const T* __restrict__ g, const T* __restrict__ x,
                                                      const float* __restrict__ mean,
                                                      const float* __restrict__ rstd,
                                                      float* __restrict__ parts, int64_t rows, int64_t D) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= D) return;
  double aw = 0., ab = 0.;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float gg = (float)g[row * D + col];
    aw += (double)gg * (double)(((float)x[row * D + col] - mean[row]) * rstd[row]);
    ab += (double)gg;
  }
  parts[((int64_t)blockIdx.y * 2) * D + col] = (float)aw;
  parts[((int64_t)blockIdx.y * 2 + 1) * D + col] = (float)ab;
}

template <typename W>
__global__ __launch_bounds__(256) void zero_kernel(W* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = (W)0.f;
}

// ------------------------------------------------------------------------------- host side
struct Shape {
  int lanes, ne;   // 0: longer than a workgroup keeps
};

// The fewest lanes that hold a row (N = elements in 16 bytes).  A lane keeps up to 32 elements
// forward, so that rows of 2048 need no exchange between waves (36064 x 2048 bf16: 68 us); backward
// keeps five values for each, and 32 of them leave one wave per SIMD (114 us instead of 93).
Shape shape_for(int64_t D, int N, bool backward) {
  for (int lanes = 8; lanes <= 64; lanes *= 2)
    if (D <= lanes * N) return {lanes, N};
  for (int ne = 2 * N; ne <= (backward ? 16 : 32); ne *= 2)
    if (D <= 64 * ne) return {64, ne};
  for (int lanes = 128; lanes <= 1024; lanes *= 2)
    if (D <= lanes * 16) return {lanes, 16};
  return {0, 0};
}

int groups_per_block(Shape s) { return s.lanes > 64 ? 1 : 256 / s.lanes; }

int parts_for(int64_t rows, int64_t D, int N) {
  const Shape s = shape_for(D, N, true);
  const int g = s.lanes ? groups_per_block(s) : 1, most = s.lanes ? kMaxParts : 64;
  const int64_t blocks = (rows + g - 1) / g;
  return (int)(blocks < most ? blocks : most);
}

// f(lanes, ne as constants) for the shapes shape_for() gives
template <int L, int E>
struct Cfg {
  static constexpr int lanes = L, ne = E, threads = L > 64 ? L : 256, groups = threads / L;
};
template <int N, bool BACKWARD, typename F>
int for_shape(Shape s, F f) {
  switch (s.lanes) {
    case 8: return f(Cfg<8, N>());
    case 16: return f(Cfg<16, N>());
    case 32: return f(Cfg<32, N>());
    case 64:
      if (s.ne == N) return f(Cfg<64, N>());
      if (s.ne == 8) return f(Cfg<64, 8>());
      if (s.ne == 16) return f(Cfg<64, 16>());
      if constexpr (!BACKWARD) return f(Cfg<64, 32>());
      return MN_EUNSUPPORTED;
    case 128: return f(Cfg<128, 16>());
    case 256: return f(Cfg<256, 16>());
    case 512: return f(Cfg<512, 16>());
    default: return f(Cfg<1024, 16>());
  }
}

template <typename T, typename W>
int fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows,
        int64_t D, float eps, hipStream_t st) {
  const float dim = (float)D;
  const Shape s = shape_for(D, Vec16<T>::N, false);
  if (!s.lanes) {
    if (rows > kLongRows) return MN_EUNSUPPORTED;
    ln_fwd_long_kernel<T, W><<<(unsigned)rows, kLongThreads, 0, st>>>(
        (const T*)x, (const W*)w, (const W*)b, (T*)y, mean, rstd, D, (double)D, eps);
    return mn_launch_status();
  }
  return for_shape<Vec16<T>::N, false>(s, [&](auto cfg) {
    using C = decltype(cfg);
    const int64_t want = (rows + C::groups - 1) / C::groups;
    const unsigned grid = (unsigned)(want < kMaxBlocks ? want : kMaxBlocks);
    ln_fwd_kernel<T, W, C::lanes, C::ne><<<grid, C::threads, 0, st>>>(
        (const T*)x, (const W*)w, (const W*)b, (T*)y, mean, rstd, rows, D, dim, eps);
    return mn_launch_status();
  });
}

template <typename T, typename W>
int bwd(const void* g, const void* x, const float* mean, const float* rstd, const void* w, void* dx,
        void* dw, void* db, int64_t rows, int64_t D, float* parts, hipStream_t st) {
  const float dim = (float)D;
  const Shape s = shape_for(D, Vec16<T>::N, true);
  int nparts = 0;
  if (!s.lanes) {
    if (rows > kLongRows) return MN_EUNSUPPORTED;
    // (before dx, which may take the gradient's place)
    if (dw || db) {
      nparts = parts_for(rows, D, Vec16<T>::N);
      ln_cols_kernel<T><<<dim3((unsigned)((D + 255) / 256), (unsigned)nparts), 256, 0, st>>>(
          (const T*)g, (const T*)x, mean, rstd, parts, rows, D);
    }
    if (dx)
      ln_bwd_long_kernel<T, W><<<(unsigned)rows, kLongThreads, 0, st>>>(
          (const T*)g, (const T*)x, mean, rstd, (const W*)w, (T*)dx, D, (double)D);
  } else {
    const int rc = for_shape<Vec16<T>::N, true>(s, [&](auto cfg) {
      using C = decltype(cfg);
      const int64_t want = (rows + C::groups - 1) / C::groups;
      const int most = parts_for(rows, D, Vec16<T>::N);
      const unsigned grid = (unsigned)(want < most ? want : most);
      const bool join = grid > 1 && (dw || db);
      nparts = join ? (int)grid : 0;
      ln_bwd_kernel<T, W, C::lanes, C::ne><<<grid, C::threads, 0, st>>>(
          (const T*)g, (const T*)x, mean, rstd, (const W*)w, (T*)dx, join ? parts : nullptr,
          join ? nullptr : (W*)dw, join ? nullptr : (W*)db, rows, D, dim);
      return mn_launch_status();
    });
    if (rc != MN_OK) return rc;
  }
  if (nparts) {
    const int64_t blocks = (D + 31) / 32;
    ln_join_kernel<W><<<dim3((unsigned)(blocks < kJoinBlocks ? blocks : kJoinBlocks), 2), 1024, 0, st>>>(
        parts, (W*)dw, (W*)db, nparts, D);
  }
  return mn_launch_status();
}

// f(element type, weight type): a weight has the rows' type or is fp32
template <typename F>
int for_types(int dtype, int wdtype, F f) {
  return mn_for_dtype(dtype, [&](auto t) {
    if (wdtype == dtype) return f(t, t);
    if (wdtype == MN_F32) return f(t, float());
    return (int)MN_EUNSUPPORTED;
  });
}

int check(int64_t rows, int64_t D) {
  if (rows < 0 || D <= 0) return MN_EINVAL;
  if (D >= (1ll << 30) || rows >= (1ll << 40) || (rows && D > (1ll << 60) / rows)) return MN_EUNSUPPORTED;
  return MN_OK;
}

}  // namespace

extern "C" {

int mn_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                      int64_t rows, int64_t D, double eps, int dtype, int wdtype, mn_stream_t stream) {
  const int st = check(rows, D);
  if (st != MN_OK) return st;
  return for_types(dtype, wdtype, [&](auto t, auto wt) {
    if (rows == 0) return (int)MN_OK;
    if (!x || !y) return (int)MN_EINVAL;
    return fwd<decltype(t), decltype(wt)>(x, w, b, y, mean, rstd, rows, D, (float)eps, mn_stream(stream));
  });
}

size_t mn_layer_norm_ws_bytes(int64_t rows, int64_t D) {
  if (check(rows, D) != MN_OK || rows == 0) return 0;
  const int a = parts_for(rows, D, 4), b = parts_for(rows, D, 8);   // enough for either width
  return (size_t)(a > b ? a : b) * 2 * (size_t)D * sizeof(float);
}

int mn_layer_norm_bwd(const void* grad, const void* x, const float* mean, const float* rstd,
                      const void* w, void* dx, void* dw, void* db, int64_t rows, int64_t D, int dtype,
                      int wdtype, void* ws, size_t ws_bytes, mn_stream_t stream) {
  const int st = check(rows, D);
  if (st != MN_OK) return st;
  return for_types(dtype, wdtype, [&](auto t, auto wt) {
    using W = decltype(wt);
    hipStream_t s = mn_stream(stream);
    if (rows == 0) {   // sums over no rows
      const unsigned grid = (unsigned)((D + 255) / 256);
      if (dw) zero_kernel<W><<<grid, 256, 0, s>>>((W*)dw, D);
      if (db) zero_kernel<W><<<grid, 256, 0, s>>>((W*)db, D);
      return mn_launch_status();
    }
    if (!grad || !x || !mean || !rstd) return (int)MN_EINVAL;
    if ((dw || db) && (!ws || ws_bytes < mn_layer_norm_ws_bytes(rows, D) || !mn_aligned(ws, 4)))
      return (int)MN_EINVAL;
    return bwd<decltype(t), W>(grad, x, mean, rstd, w, dx, dw, db, rows, D, (float*)ws, s);
  });
}

}  // extern "C"
