// Attention over a sliding window plus a few first tokens ("sinks"), forward and backward, for
// training: queries and keys of one sequence of T tokens, heads of queries sharing heads of keys.
//
//   visible(i, j):  j <= i + right  and  (j >= i - left  or  j < sinks)  and  i, j < length
//   P = softmax_j(scale q_i k_j),  o = P v,  lse = log sum_j exp(scale q_i k_j)
//   dv = P^T do,  dP = do v^T,  dS = P (dP - rowsum(do o)),  dq = scale dS k,  dk = scale dS^T q
//
// Scores are never stored: forward keeps a running maximum and sum per row, backward computes P
// again from lse.  All products run on the matrix cores with fp32 accumulators: 16-bit types on
// 32x32x16 instructions, fp32 on 32x32x2.
//
// Orientation.  A 32x32 accumulator holds one COLUMN per lane (lane l: column l % 32, of its 32
// rows the 16 with bit 2 equal to l / 32).  Scores are computed transposed where a row of the
// softmax runs over keys (S^T = K Q^T: a lane owns one query, so maximum and sum are a fold over
// registers and one swap with lane l ^ 32), and the accumulator's registers are, in order,
// the B operand of the next product over the same 32 keys (or queries): which of the 32 a slot of
// the contraction means is free as long as A uses the same assignment, and the A operand is read
// from LDS for exactly those.  P and dS therefore never leave the registers of their lane.
//
// LDS tiles hold rows of D elements as they lie in memory; 16-byte chunk c of row r is stored at
// chunk c ^ swz(r), which spreads both kinds of reads over all banks: rows (a lane reads 16 bytes
// of its row) and transposed (16-bit: ds_read_b64_tr_b16 gives a lane four rows' values of its
// column; fp32: plain 4-byte reads).  Two buffers of two tiles: 64 KB at D = 128, two workgroups a
// CU; rows of whole 16-byte chunks go from memory to LDS without registers, others through them:
// 2.3 to 2.8 times slower (batch 2 of 16 heads, 4099 tokens, causal, bf16: D = 104 and 100 forward
// 196 and 492 us, backward 666 and 1519 us; 128 and 127: 202 and 553, 672 and 1732 us).  Through
// registers, 16-bit types spill 25 of them in dk / dv and 4 in dq at D = 97 .. 128.
//
// Measured at T = 4099, causal, batch 8 of 16 heads, D = 128, bf16 (operations a visible pair needs
// over time; a large bf16 matrix product of the library runs at 1160 TFLOP/s): forward 0.67 ms, 820
// TFLOP/s; dq 0.89 ms, 925; dk and dv 1.54 ms, 716 (of the 8 D they need; they run 10 D).  The
// matrix cores are busy 0.37, 0.43 and 0.41 of the time, LDS a sixth of it without conflicts: what is
// left are waits of two waves per SIMD for LDS, for each other's products and at the barrier of a
// tile.  fp32: 33 % to 60 % of the 154 TFLOP/s of a library product.
//
// Tried and not kept: 16 instead of 32 columns a wave (half the registers, twice the LDS reads: dk
// and dv together at D = 128 in 0.62 ms where 32-wide halves take 0.50); dk and dv in one workgroup
// (one wave per SIMD or spills: 0.98 ms); two waves sharing a wave's rows where there are few
// workgroups (a CU's matrix cores have the same work: 24 us instead of 25 at batch 8, 197 tokens,
// fp32); the row sums as a product with ones (no faster, and lse would carry P's rounding); four
// waves per SIMD instead of three at D = 64 (11 x 988 tokens: 48 us either way); the four waves of a
// workgroup of sinks alone taking turns with its queries (15808 tokens: no faster, and spills).
#include <mutex>
#include <type_traits>

#include "elem.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / MN_WAVE;
constexpr int kMaxD = 128;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Args {
  const void *q, *k, *v, *out, *grad;   // out, grad: dense [B, T, Hq, D]
  void *o, *dq, *dk, *dv;               // dense results
  float *lse;                           // [B, Hq, T]
  float *delta;                         // [B, Hq, T] rowsum(do * o), written by the dq kernel
  float *parts;                         // partial dk, dv of key tiles that are split over queries
  const int32_t* lengths;
  int64_t sq[3], sk[3], sv[3];          // strides of b, t, h in elements
  int32_t T, Hq, Hkv, D, left, right, sinks;
  int32_t tiles, group;
  int32_t sink_tiles, sink_rows, chunk, nchunks;   // dk / dv: see there
  int32_t fold;                         // tiles differ in work: see tile_of
  float scale, scale_log2;
};

// ------------------------------------------------------------------------- matrix-core types
template <typename T>
struct Mma;
template <>
struct Mma<bf16_t> {
  typedef bf16_t frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<f16_t> {
  typedef f16_t frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {   // four contraction slots a lane: four instructions of two
  typedef float frag __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes a lane from memory (uniform address + 32-bit offset) to LDS (wave-uniform address +
// 16 * lane), asynchronous: the data is there after wait_loads() and a barrier.  In assembly
// because the compiler, which cannot tell the two buffers apart, would wait for the load before
// the next read of LDS; m0 is put back.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t offset, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(m0)
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(base)
               : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// The order of a block of N products, each fed by READS reads of LDS: reads run AHEAD products
// before their use.  (Left alone, the compiler reads right before each product and waits.)
template <int N, int READS, int AHEAD>
__device__ __forceinline__ void feed() {
  constexpr int kMfma = 0x8, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, READS * AHEAD, 0);
#pragma unroll
  for (int k = 0; k < N - AHEAD; ++k) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, AHEAD, 0);
}
// One tile of rows in LDS: DP elements a row (D rounded up to 32, zeros behind D).
template <typename T, int DP, int ROWS>
struct Tile {
  typedef typename Mma<T>::frag frag;
  static constexpr int N = 16 / (int)sizeof(T);      // elements of a chunk
  static constexpr int CH = DP / N;                  // chunks of a row that hold data
  static constexpr int NC = CH <= 4 ? 4 : CH <= 8 ? 8 : CH <= 16 ? 16 : 32;   // chunks of a row
  static constexpr int STEPS = CH / 2;               // steps of a contraction over D
  static constexpr int BYTES = ROWS * NC * 16;
  static constexpr int PER = ROWS * CH / kThreads;   // chunks a thread stages
  static_assert(ROWS * CH % kThreads == 0 && ROWS * NC % kThreads == 0, "whole chunks per thread");

  static __device__ __forceinline__ int swz(int row) {
    if (NC >= 16) return (row & 3) << 2 | (row >> 2 & 3);
    if (NC == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    return row >> 2 & 3;
  }
  static __device__ __forceinline__ int at(int row, int chunk) {
    return (row * NC + (chunk ^ swz(row))) * 16;
  }

  // global -> registers: the tile's rows from `rows` on, zeros from row `left` on
  static __device__ __forceinline__ void fetch(frag* regs, const T* rows, int64_t stride, int left, int D) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int idx = threadIdx.x + p * kThreads, row = idx / CH, col = idx % CH * N;
      regs[p] = chunk(rows + row * stride + col, row < left ? D - col : 0, D);
    }
  }
  // `cnt` elements of a row from p on, zeros behind them.  The end of a row of at least N elements
  // is taken from the 16 bytes that end there, moved down: one load, no loop over elements.
  static __device__ __forceinline__ frag chunk(const T* p, int cnt, int D) {
    if (cnt <= 0) return (frag)(0.f);
    if (D >= N) {
      const int missing = max(N - cnt, 0);
      typedef uint64_t half2 __attribute__((ext_vector_type(2)));
      half2 v = __builtin_bit_cast(half2, *reinterpret_cast<const typename Vec16<T>::utype*>(p - missing));
      if (missing) {
        const int bits = missing * 8 * (int)sizeof(T);   // 16 .. 112
        const uint64_t lo = bits < 64 ? v[0] >> bits | v[1] << (64 - bits) : v[1] >> (bits - 64);
        v[1] = bits < 64 ? v[1] >> bits : 0;
        v[0] = lo;
      }
      return __builtin_bit_cast(frag, v);
    }
    frag f;
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = e < cnt ? p[e] : (T)0.f;
    return f;
  }
  static __device__ __forceinline__ void put(char* lds, const frag* regs) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int idx = threadIdx.x + p * kThreads;
      *reinterpret_cast<frag*>(lds + at(idx / CH, idx % CH)) = regs[p];
    }
  }
  // global -> LDS without registers: the memory system writes 16 bytes per lane, 1 KB per wave and
  // instruction in the order of the lanes, so the swizzle is in which chunk a lane asks for.
  // Rows from `end` on repeat the last one: what is multiplied with them is zero.  Needs
  // 16-byte aligned rows of whole chunks; chunks behind D are not written (see clear).
  static constexpr int SLOTS = ROWS * NC / kThreads;
  static __device__ __forceinline__ uint32_t offset(int p, int rows, int64_t stride) {
    const int slot = threadIdx.x + p * kThreads, row = min(slot / NC, rows - 1), chunk = slot % NC ^ swz(slot / NC);
    return (uint32_t)((row * stride + chunk * N) * (int)sizeof(T));
  }
  // `offsets`: those of a whole tile, which a thread keeps
  static __device__ __forceinline__ void load(uint32_t lds, const T* rows, const uint32_t* offsets, int64_t stride,
                                              int left, int D) {
    if (__builtin_expect(left < ROWS, 0)) {
      asm volatile("");   // (a branch, not both sides)
      uint32_t cut[SLOTS];
#pragma unroll
      for (int p = 0; p < SLOTS; ++p) cut[p] = offset(p, left, stride);
      load_all(lds, rows, cut, D);
    } else {
      load_all(lds, rows, offsets, D);
    }
  }
  static __device__ __forceinline__ void load_all(uint32_t lds, const T* rows, const uint32_t* offsets, int D) {
#pragma unroll
    for (int p = 0; p < SLOTS; ++p) {
      const int slot = threadIdx.x + p * kThreads, chunk = slot % NC ^ swz(slot / NC);
      const uint32_t at = lds + (p * kThreads + (threadIdx.x & ~(MN_WAVE - 1))) * 16;
      if (D == NC * N || chunk * N < D) load_to_lds((const char*)rows, offsets[p], at);
    }
  }
  static __device__ __forceinline__ void clear(char* lds, int D) {
    if (D == NC * N) return;
#pragma unroll
    for (int p = 0; p < ROWS * NC / kThreads; ++p) {
      const int slot = threadIdx.x + p * kThreads, row = slot / NC, chunk = slot % NC ^ swz(row);
      if (chunk * N >= D) *reinterpret_cast<frag*>(lds + slot * 16) = (frag)(0.f);
    }
  }
  // A operand whose row is the lane's (row0 + l % 32), step s of a contraction over D
  static __device__ __forceinline__ frag rows(const char* lds, int row0, int s) {
    const int lane = threadIdx.x % MN_WAVE;
    return *reinterpret_cast<const frag*>(lds + at(row0 + lane % 32, 2 * s + lane / 32));
  }
  // A operand whose row is column d0 + l % 32 of the tile, step s of a contraction over the 32
  // rows from row0 on, in the order of an accumulator's registers
  static __device__ __forceinline__ frag cols(const char* lds, int row0, int s, int d0) {
    const int lane = threadIdx.x % MN_WAVE, half = lane / 32;
    frag f;
    if constexpr (sizeof(T) == 2) {
      const int i = lane % 16, d = d0 + lane % 32 / 16 * 16 + i % 4 * 4;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int row = row0 + 16 * s + 8 * g + 4 * half + i / 4;
        const char* p = lds + at(row, d / 8) + d % 8 * 2;
        typedef T quad __attribute__((ext_vector_type(4)));
        const quad v = __builtin_bit_cast(quad, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * g + e] = v[e];
      }
    } else {
      const int d = d0 + lane % 32;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = row0 + 8 * s + 4 * half + e;
        f[e] = *reinterpret_cast<const T*>(lds + at(row, d / 4) + d % 4 * 4);
      }
    }
    return f;
  }
};

// Two buffers of two tiles (keys and values, or queries and gradients): while one is multiplied,
// the other is filled, straight from memory if DIRECT, through registers otherwise.
template <typename T, int DP, int ROWS, bool DIRECT, int EXTRA>
struct Stage {
  typedef Tile<T, DP, ROWS> Ti;
  static constexpr int kBuf = 2 * Ti::BYTES + EXTRA;
  char* lds;
  typename Ti::frag r0[DIRECT ? 1 : Ti::PER], r1[DIRECT ? 1 : Ti::PER];
  uint32_t o0[DIRECT ? Ti::SLOTS : 1], o1[DIRECT ? Ti::SLOTS : 1];

  __device__ __forceinline__ char* buffer(int n) const { return lds + (n & 1) * kBuf; }
  __device__ __forceinline__ void init(char* p, int64_t sa, int64_t sb, int D) {
    lds = p;
    if constexpr (DIRECT) {
#pragma unroll
      for (int k = 0; k < Ti::SLOTS; ++k) {
        o0[k] = Ti::offset(k, ROWS, sa);
        o1[k] = Ti::offset(k, ROWS, sb);
      }
      for (int n = 0; n < 2; ++n) {
        Ti::clear(buffer(n), D);
        Ti::clear(buffer(n) + Ti::BYTES, D);
      }
    }
  }
  // tile n: rows of two heads from a and b on, `left` of them there
  __device__ __forceinline__ void begin(int n, const T* a, int64_t sa, const T* b, int64_t sb, int left, int D) {
    if constexpr (DIRECT) {
      const uint32_t at = lds_address(buffer(n));
      Ti::load(at, a, o0, sa, left, D);
      Ti::load(at + Ti::BYTES, b, o1, sb, left, D);
    } else {
      Ti::fetch(r0, a, sa, left, D);
      Ti::fetch(r1, b, sb, left, D);
    }
  }
  __device__ __forceinline__ void finish(int n) {
    if constexpr (DIRECT) {
      wait_loads();
    } else {
      Ti::put(buffer(n), r0);
      Ti::put(buffer(n) + Ti::BYTES, r1);
    }
  }
};

// Steps of a contraction over an accumulator's 32 rows, and the B operand of one of them: the
// registers in order, rounded to T once (16-bit types: P in [0, 1] and dS carry 2^-8 or 2^-11 of
// themselves, the rounding the result gets anyway; the sums stay fp32).
template <typename T>
struct Acc {
  static constexpr int N = 16 / (int)sizeof(T);
  static constexpr int STEPS = 16 / N;
  static __device__ __forceinline__ typename Mma<T>::frag operand(const f32x16& a, int s) {
    typename Mma<T>::frag f;
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (T)a[s * N + e];
    return f;
  }
};

// Row of an accumulator's register r, less the 4 of a lane of the upper half.
__device__ __forceinline__ constexpr int acc_row(int r) { return r / 4 * 8 + r % 4; }

// In a branch few tiles take: keeps the compiler from computing both sides for all of them.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// What a lane's query sees of a tile, or which of a tile's queries see a lane's key, for the row
// numbers of an accumulator (constants c = r / 4 * 8 + r % 4; the lane's half is in the bounds):
// one interval, and the first few.
struct Seen {
  int lo, first;
  unsigned span;
  __device__ __forceinline__ bool operator()(int c) const { return (unsigned)(c - lo) <= span || c < first; }
};
__device__ __forceinline__ Seen interval(int lo, int hi, int first, int row0) {
  const int base = row0 + (int)(threadIdx.x % MN_WAVE / 32) * 4;
  if (hi < lo) return {1 << 30, first - base, 0u};
  return {lo - base, first - base, (unsigned)(hi - lo)};
}
// keys of query i in the tile that starts at j0 (sinks end where the others do)
__device__ __forceinline__ Seen keys_seen(const Args& a, int i, int j0, int len) {
  const int hi = min(i + a.right, len - 1);
  return interval(max(i - a.left, 0), hi, min(a.sinks, hi + 1), j0);
}

// Where the keys of queries q0 .. q1 lie: tiles [0, sinks) and [first, last) of ROWS keys.
struct KeyTiles {
  int sinks, first, last;
  __device__ __forceinline__ int count() const { return sinks + last - first; }
  __device__ __forceinline__ int tile(int n) const { return n < sinks ? n : first + n - sinks; }
};
template <int ROWS>
__device__ __forceinline__ KeyTiles key_tiles(const Args& a, int q0, int q1, int len) {
  const int lo = max(0, q0 - a.left), hi = min(len - 1, q1 + a.right);
  KeyTiles t;
  t.first = lo / ROWS;
  t.last = hi / ROWS + 1;
  t.sinks = min((min(a.sinks, len) + ROWS - 1) / ROWS, t.first);
  return t;
}

// Does every one of the queries q0 .. q1 see all keys k0 .. k1, does any see any of them?
__device__ __forceinline__ bool all_visible(const Args& a, int q0, int q1, int k0, int k1, int len) {
  return k1 < len && k1 <= q0 + a.right && (k0 >= q1 - a.left || k1 < a.sinks);
}
__device__ __forceinline__ bool none_visible(const Args& a, int q0, int q1, int k0, int k1) {
  return k0 > q1 + a.right || (k1 < q0 - a.left && k0 >= a.sinks);
}

__device__ __forceinline__ int length_of(const Args& a, int b) {
  if (!a.lengths) return a.T;
  return min(max(a.lengths[b], 0), a.T);
}

// B operands of a lane's own row (query or key) straight from memory; `valid` false: zeros.
template <typename T, int DP>
__device__ __forceinline__ void own_row(typename Mma<T>::frag* f, const T* row, bool valid, int D) {
  typedef Tile<T, DP, 64> Ti;
  const int half = threadIdx.x % MN_WAVE / 32;
#pragma unroll
  for (int s = 0; s < Ti::STEPS; ++s) {
    const int col = (2 * s + half) * Ti::N;
    f[s] = Ti::chunk(row + col, valid ? D - col : 0, D);
  }
}

// A transposed accumulator (rows = elements of a head, column = the lane's token) to its row,
// times `factor`; factor 0 (a token behind the end): zeros, whatever was accumulated.
template <typename T, int DP>
__device__ __forceinline__ void store_columns(T* row, const f32x16* acc, float factor, int D) {
  typedef T quad __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const int half = threadIdx.x % MN_WAVE / 32;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + g * 8 + half * 4;
      if (d + 4 <= D) {
        quad v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = factor == 0.f ? (T)0.f : (T)(acc[db][4 * g + e] * factor);
        *reinterpret_cast<quad*>(row + d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) row[d + e] = factor == 0.f ? (T)0.f : (T)(acc[db][4 * g + e] * factor);
      }
    }
}

// Which tile of which head (counting the batch) a workgroup has.  Each of the 8 XCDs runs a
// contiguous range of (key head, tile, query head), so that neighbours find each other's keys in
// its L2 (T = 15808, window 1024, 4 heads to a key head: forward reads 304 MB past the L2 with the
// query heads one after the other, 100 side by side).  Where tiles differ in work (one side of the
// window open beyond a quarter of the sequence), `fold`: query heads follow each other, and a head's
// tiles are taken in pairs from both ends, which gives any range the same share of long and short
// ones; a range runs its long ones first.  Folded against not, us forward / backward, causal, 16 heads
// on 4 of D = 128, bf16:
//   15808 tokens   window T/16: 179/602, 170/601   T/4: 508/2001, 522/2039   none: 1108/4535, 1373/5590
//   8 x 2048       window T/16: 74/203, 74/204     T/4: 104/354, 98/346      none: 178/694, 184/743
//   2 x 4099       window T/16: 48/156, 44/125     T/4: 86/333, 87/308       none: 191/765, 183/756
// (T/4 is where the long sequence starts to win; few workgroups lose up to 8 % by it.)
struct TileOf {
  int tile, head;
};
__device__ __forceinline__ TileOf tile_of(const Args& a, int tiles, int group, bool last_is_long) {
  if (!a.fold) {
    const uint32_t slot = xcd_slot(), k = slot / group;
    return {(int)(k % tiles), (int)(k / tiles * group + slot % group)};
  }
  const uint32_t total = gridDim.x, xcd = blockIdx.x & 7u, j = blockIdx.x >> 3, rem = total & 7u;
  const uint32_t start = xcd * (total >> 3) + (xcd < rem ? xcd : rem), n = (total >> 3) + (xcd < rem ? 1 : 0);
  const uint32_t half = (n + 1) / 2, slot = start + (j < half ? 2 * j : 2 * (j - half) + 1);
  const int k = slot % tiles, from_front = k & 1 ? tiles - 1 - k / 2 : k / 2;
  return {last_is_long ? tiles - 1 - from_front : from_front, (int)(slot / tiles)};
}

// What the registers allow (fp32 at D > 64: operands and accumulators need more than 256).
template <typename T, int DP>
constexpr int kWavesPerSimd = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
// Rows of keys in a tile: fp32 rows are twice as long.
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 64 : 32;
constexpr int kQueries = 32 * kWaves;   // queries (or, for dk / dv, keys) of a workgroup

// --------------------------------------------------------------------------------- forward
template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads, (kWavesPerSimd<T, DP>)) void attn_fwd_kernel(const Args a) {
  constexpr int R = kRows<T>, KT = R / 32;
  typedef Tile<T, DP, R> Ti;
  typedef typename Mma<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const TileOf me = tile_of(a, a.tiles, a.group, a.left > a.right);
  const int tile = me.tile, h = me.head % a.Hq, b = me.head / a.Hq;
  const int len = length_of(a, b);
  const int wave = threadIdx.x / MN_WAVE, lane = threadIdx.x % MN_WAVE;
  const int q0 = tile * kQueries, w0 = q0 + wave * 32, i = w0 + lane % 32;
  T* orow = (T*)a.o + (((int64_t)b * a.T + i) * a.Hq + h) * a.D;
  float* lse = a.lse + ((int64_t)b * a.Hq + h) * a.T;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = (f32x16)(0.f);
  float m = -INFINITY, sum = 0.f;
  if (q0 < len) {
    frag qf[Ti::STEPS];
    own_row<T, DP>(qf, (const T*)a.q + b * a.sq[0] + h * a.sq[2] + i * a.sq[1], i < len, a.D);
    const T* kb = (const T*)a.k + b * a.sk[0] + h / a.group * a.sk[2];
    const T* vb = (const T*)a.v + b * a.sv[0] + h / a.group * a.sv[2];
    const KeyTiles kt = key_tiles<R>(a, q0, min(q0 + kQueries, len) - 1, len);
    const int n_tiles = kt.count(), w1 = min(w0 + 31, len - 1);
    Stage<T, DP, R, DIRECT, 0> stage;
    stage.init(lds, a.sk[1], a.sv[1], a.D);
    const auto begin = [&](int n) {
      const int row0 = kt.tile(n) * R;
      stage.begin(n, kb + row0 * a.sk[1], a.sk[1], vb + row0 * a.sv[1], a.sv[1], len - row0, a.D);
    };
    begin(0);
    for (int n = 0; n < n_tiles; ++n) {
      const char* kl = stage.buffer(n);
      const char* vl = kl + Ti::BYTES;
      stage.finish(n);
      __syncthreads();   // (everyone is done with the other buffer)
      if (n + 1 < n_tiles) begin(n + 1);
      const int j0 = kt.tile(n) * R;
      if (w0 >= len || none_visible(a, w0, w1, j0, j0 + R - 1)) continue;
      f32x16 s[KT];
      float top = -INFINITY;
      const bool whole = all_visible(a, w0, w1, j0, j0 + R - 1, len);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        s[t] = (f32x16)(0.f);
#pragma unroll
        for (int st = 0; st < Ti::STEPS; ++st) s[t] = Mma<T>::mul(Ti::rows(kl, t * 32, st), qf[st], s[t]);
        if constexpr (sizeof(T) == 2) feed<Ti::STEPS, 1, 4 < Ti::STEPS ? 4 : Ti::STEPS>();
        if (!whole) {
          keep_branch();
          const Seen see = keys_seen(a, i, j0 + t * 32, len);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = see(acc_row(r)) ? s[t][r] : -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
      }
      top = max_xor32(top) * a.scale_log2;
      // a new maximum only where the old one is left behind by more than 2^8: below that P stays
      // below 2^8 and nothing has to be scaled
      if (__builtin_expect(__any(top > m + 8.f), 0)) {
        const float now = fmaxf(m, top), f = now == -INFINITY ? 1.f : exp2f(m - now);
        m = now;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= f;
      }
      const float base = m == -INFINITY ? 0.f : m;   // nothing seen yet: exp2(-inf - 0) = 0
#pragma unroll
      for (int t = 0; t < KT; ++t) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale_log2, -base));
          sum += s[t][r];
        }
#pragma unroll
        for (int st = 0; st < Acc<T>::STEPS; ++st) {
          const frag p = Acc<T>::operand(s[t], st);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
            acc[d] = Mma<T>::mul(Ti::cols(vl, t * 32, st, d * 32), p, acc[d]);
        }
      }
    }
  }
  if (i >= a.T) return;
  sum = plus_xor32(sum);
  const bool any = i < len && m != -INFINITY;   // (a NaN among the scores: m may be -inf, sum is NaN)
  const bool valid = i < len && (any || sum != sum);
  store_columns<T, DP>(orow, acc, valid ? 1.f / sum : 0.f, a.D);
  if (lane < 32) lse[i] = valid ? (m + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
}

// -------------------------------------------------------------- backward: dq (and rowsum(do o))
template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads, (kWavesPerSimd<T, DP>)) void attn_dq_kernel(const Args a) {
  constexpr int R = kRows<T>, KT = R / 32;
  typedef Tile<T, DP, R> Ti;
  typedef typename Mma<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const TileOf me = tile_of(a, a.tiles, a.group, a.left > a.right);
  const int tile = me.tile, h = me.head % a.Hq, b = me.head / a.Hq;
  const int len = length_of(a, b);
  const int wave = threadIdx.x / MN_WAVE, lane = threadIdx.x % MN_WAVE;
  const int q0 = tile * kQueries, w0 = q0 + wave * 32, i = w0 + lane % 32;
  const int64_t row = (((int64_t)b * a.T + i) * a.Hq + h) * a.D;
  const int64_t stat = ((int64_t)b * a.Hq + h) * a.T + i;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = (f32x16)(0.f);
  if (q0 < len) {
    frag qf[Ti::STEPS], gf[Ti::STEPS];
    own_row<T, DP>(qf, (const T*)a.out + row, i < len, a.D);
    own_row<T, DP>(gf, (const T*)a.grad + row, i < len, a.D);
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < Ti::STEPS; ++s)
#pragma unroll
      for (int e = 0; e < Ti::N; ++e) delta += (float)qf[s][e] * (float)gf[s][e];
    delta = plus_xor32(delta);
    if (i < len && lane < 32) a.delta[stat] = delta;
    const float l2 = i < len ? a.lse[stat] * kLog2e : INFINITY;   // no query: P = exp2(-inf) = 0
    own_row<T, DP>(qf, (const T*)a.q + b * a.sq[0] + h * a.sq[2] + i * a.sq[1], i < len, a.D);
    const T* kb = (const T*)a.k + b * a.sk[0] + h / a.group * a.sk[2];
    const T* vb = (const T*)a.v + b * a.sv[0] + h / a.group * a.sv[2];
    const KeyTiles kt = key_tiles<R>(a, q0, min(q0 + kQueries, len) - 1, len);
    const int n_tiles = kt.count(), w1 = min(w0 + 31, len - 1);
    Stage<T, DP, R, DIRECT, 0> stage;
    stage.init(lds, a.sk[1], a.sv[1], a.D);
    const auto begin = [&](int n) {
      const int row0 = kt.tile(n) * R;
      stage.begin(n, kb + row0 * a.sk[1], a.sk[1], vb + row0 * a.sv[1], a.sv[1], len - row0, a.D);
    };
    begin(0);
    for (int n = 0; n < n_tiles; ++n) {
      const char* kl = stage.buffer(n);
      const char* vl = kl + Ti::BYTES;
      stage.finish(n);
      __syncthreads();
      if (n + 1 < n_tiles) begin(n + 1);
      const int j0 = kt.tile(n) * R;
      if (w0 >= len) continue;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const int jt = j0 + t * 32;
        if (none_visible(a, w0, w1, jt, jt + 31)) continue;
        f32x16 s = (f32x16)(0.f), p = (f32x16)(0.f);
#pragma unroll
        for (int st = 0; st < Ti::STEPS; ++st) {
          s = Mma<T>::mul(Ti::rows(kl, t * 32, st), qf[st], s);
          p = Mma<T>::mul(Ti::rows(vl, t * 32, st), gf[st], p);
        }
        if constexpr (sizeof(T) == 2) feed<2 * Ti::STEPS, 1, 4>();
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -l2)) * (p[r] - delta);
        if (!all_visible(a, w0, w1, jt, jt + 31, len)) {
          keep_branch();
          const Seen see = keys_seen(a, i, jt, len);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = see(acc_row(r)) ? s[r] : 0.f;
        }
#pragma unroll
        for (int st = 0; st < Acc<T>::STEPS; ++st) {
          const frag ds = Acc<T>::operand(s, st);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
            acc[d] = Mma<T>::mul(Ti::cols(kl, t * 32, st, d * 32), ds, acc[d]);
        }
        if constexpr (sizeof(T) == 2) feed<Acc<T>::STEPS * DP / 32, 2, 2>();
      }
    }
  }
  if (i < a.T) store_columns<T, DP>((T*)a.dq + row, acc, i < len ? a.scale : 0.f, a.D);
}

// -------------------------------------------------------------------- backward: dk and dv
// A workgroup owns 128 keys, a wave 32 of them as columns, and walks over the queries that see
// them, for every query head of the group in turn, so a shared head's gradient is one sum in
// registers, in a fixed order.
// dk and dv of a tile are two workgroups, which costs the scores twice (10 D instead of 8 D
// operations a pair) and is faster: both at once are 2 x 64 accumulators and 2 x 32 registers of
// keys and values at D = 128, which leaves no room for LDS reads in flight at two waves per SIMD
// (T = 15808, window 1024, 16 heads on 4 of keys: 0.48 ms, in one workgroup 0.98).
// Key tiles that hold sinks are seen by all later queries: their queries behind the window are
// given to `nchunks` workgroups more (chunk queries each); all of a split tile's workgroups write
// fp32 partial results, which attn_join_kernel adds in order.  Without that the one workgroup of
// the sinks would run T / (left + 128) times as long as any other.
struct KeyWork {
  int tile, part;      // part 0: the window's queries, c + 1: chunk c of those behind it
  int hk, b, len, k0, lo, hi;
  bool split, is_dk;
};
__device__ __forceinline__ KeyWork key_work(const Args& a) {
  KeyWork w;
  // the extra workgroups of the sinks stand evenly between the others
  const int extra = a.sink_tiles * a.nchunks, items = a.tiles + extra;
  const TileOf me = tile_of(a, 2 * items, 1, a.right > a.left);
  const int item = me.tile / 2;
  w.is_dk = me.tile % 2 == 0;
  w.hk = me.head % a.Hkv;
  w.b = me.head / a.Hkv;
  w.len = length_of(a, w.b);
  const int before = (int)((int64_t)item * extra / items);   // extra ones before this item
  if ((int)((int64_t)(item + 1) * extra / items) > before) {
    w.tile = before / a.nchunks;
    w.part = before % a.nchunks + 1;
  } else {
    w.tile = item - before;
    w.part = 0;
  }
  w.split = w.tile < a.sink_tiles;
  w.k0 = w.tile * kQueries;
  const int k1 = min(w.k0 + kQueries, w.len) - 1;
  w.lo = max(0, w.k0 - a.right);
  w.hi = min((int64_t)w.len - 1, (int64_t)k1 + a.left);
  if (w.part > 0) {
    w.lo = min((int64_t)a.T, (int64_t)w.k0 + kQueries + a.left + (int64_t)(w.part - 1) * a.chunk);
    w.hi = min((int64_t)w.len - 1, (int64_t)w.lo + a.chunk - 1);
  } else if (w.split) {
    w.hi = min((int64_t)w.len - 1, (int64_t)w.k0 + kQueries - 1 + a.left);
  } else if (w.k0 < a.sinks) {
    w.hi = w.len - 1;
  }
  return w;
}

// The staged queries of a workgroup: tiles of R rows, head after head.
template <typename T, int DP, int R, bool DIRECT>
struct QueryTiles {
  typedef Stage<T, DP, R, DIRECT, 2 * R * (int)sizeof(float)> St;
  St stage;
  int count, row;                   // tiles; first row of the one that was finished last
  int first, head, next, pending;   // what begin() will load, what it has begun
  const T *qp, *gp;                 // rows `next` of head `head`
  const float *lp, *dp;
  float lreg = 0.f, dreg = 0.f;
  __device__ __forceinline__ void point(const Args& a, const KeyWork& w) {
    qp = (const T*)a.q + w.b * a.sq[0] + head * a.sq[2] + next * a.sq[1];
    gp = (const T*)a.grad + (((int64_t)w.b * a.T + next) * a.Hq + head) * a.D;
    const int64_t stat = ((int64_t)w.b * a.Hq + head) * a.T + next;
    lp = a.lse + stat;
    dp = a.delta + stat;
  }
  __device__ __forceinline__ void init(const Args& a, const KeyWork& w, char* lds) {
    first = next = w.lo / R * R;
    count = (w.hi / R + 1 - w.lo / R) * a.group;
    head = w.hk * a.group;
    stage.init(lds, a.sq[1], (int64_t)a.Hq * a.D, a.D);
    point(a, w);
  }
  __device__ __forceinline__ void begin(const Args& a, const KeyWork& w, int n) {
    pending = next;
    stage.begin(n, qp, a.sq[1], gp, (int64_t)a.Hq * a.D, w.len - next, a.D);
    if (threadIdx.x < R) {
      const bool there = next + (int)threadIdx.x < w.len;
      lreg = there ? lp[threadIdx.x] : INFINITY;   // no query: P = exp2(-inf) = 0
      dreg = there ? dp[threadIdx.x] : 0.f;
    }
    next += R;
    if (next > w.hi) {
      next = first;
      ++head;
      point(a, w);
    } else {
      qp += R * a.sq[1];
      gp += (int64_t)R * a.Hq * a.D;
      lp += R;
      dp += R;
    }
  }
  __device__ __forceinline__ const char* q(int n) const { return stage.buffer(n); }
  __device__ __forceinline__ const char* g(int n) const { return stage.buffer(n) + St::Ti::BYTES; }
  __device__ __forceinline__ float* stats(int n) const {   // lse in log2 units [R], delta [R]
    return reinterpret_cast<float*>(stage.buffer(n) + 2 * St::Ti::BYTES);
  }
  __device__ __forceinline__ void finish(int n) {
    stage.finish(n);
    row = pending;
    if (threadIdx.x < R) {
      stats(n)[threadIdx.x] = lreg * kLog2e;
      stats(n)[R + threadIdx.x] = dreg;
    }
  }
};

template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads, (kWavesPerSimd<T, DP>)) void attn_dkv_kernel(const Args a) {
  constexpr int R = kRows<T>;
  typedef Tile<T, DP, R> Ti;
  typedef typename Mma<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const KeyWork w = key_work(a);
  const int wave = threadIdx.x / MN_WAVE, lane = threadIdx.x % MN_WAVE;
  const int w0 = w.k0 + wave * 32, j = w0 + lane % 32, w1 = min(w0 + 31, w.len - 1);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = (f32x16)(0.f);
  if (w.k0 < w.len && w.lo <= w.hi) {
    QueryTiles<T, DP, R, DIRECT> tiles;
    tiles.init(a, w, lds);
    tiles.begin(a, w, 0);
    frag kf[Ti::STEPS];
    own_row<T, DP>(kf, (const T*)a.k + w.b * a.sk[0] + w.hk * a.sk[2] + j * a.sk[1], j < w.len, a.D);
    const auto walk = [&](auto which) {
      constexpr bool DK = decltype(which)::value;
      frag vf[DK ? Ti::STEPS : 1];
      if constexpr (DK)
        own_row<T, DP>(vf, (const T*)a.v + w.b * a.sv[0] + w.hk * a.sv[2] + j * a.sv[1], j < w.len, a.D);
      for (int n = 0; n < tiles.count; ++n) {
        const char *ql = tiles.q(n), *gl = tiles.g(n);
        const float* stats = tiles.stats(n);
        tiles.finish(n);
        __syncthreads();
        const int row0 = tiles.row;
        if (n + 1 < tiles.count) tiles.begin(a, w, n + 1);
#pragma unroll
        for (int t = 0; t < R / 32; ++t) {
          const int it = row0 + t * 32;
          // (queries outside [lo, hi] belong to another workgroup of the tile)
          if (w0 >= w.len || it > w.hi || it + 31 < w.lo || none_visible(a, it, it + 31, w0, w1)) continue;
          f32x16 s = (f32x16)(0.f), p = (f32x16)(0.f);
#pragma unroll
          for (int st = 0; st < Ti::STEPS; ++st) {
            s = Mma<T>::mul(Ti::rows(ql, t * 32, st), kf[st], s);
            if constexpr (DK) p = Mma<T>::mul(Ti::rows(gl, t * 32, st), vf[st], p);
          }
          if constexpr (sizeof(T) == 2) feed<(DK ? 2 : 1) * Ti::STEPS, 1, DK ? 4 : (Ti::STEPS < 4 ? Ti::STEPS : 4)>();
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4_t l2 = *reinterpret_cast<const float4_t*>(stats + t * 32 + g * 8 + lane / 32 * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.scale_log2, -l2[e]));
            if constexpr (DK) {
              const float4_t de = *reinterpret_cast<const float4_t*>(stats + R + t * 32 + g * 8 + lane / 32 * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[4 * g + e] *= p[4 * g + e] - de[e];
            }
          }
          if (!(it >= w.lo && it + 31 <= w.hi && all_visible(a, it, it + 31, w0, w0 + 31, w.len))) {
            keep_branch();
            const int last = j < a.sinks ? w.hi : min(w.hi, j + a.left);
            const Seen see = interval(max(w.lo, j - a.right), j < w.len ? last : -1, 0, it);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = see(acc_row(r)) ? s[r] : 0.f;
          }
#pragma unroll
          for (int st = 0; st < Acc<T>::STEPS; ++st) {
            const frag f = Acc<T>::operand(s, st);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
              acc[d] = Mma<T>::mul(Ti::cols(DK ? ql : gl, t * 32, st, d * 32), f, acc[d]);
          }
          if constexpr (sizeof(T) == 2) feed<Acc<T>::STEPS * DP / 32, 2, 2>();
        }
      }
    };
    if (w.is_dk)
      walk(std::true_type());
    else
      walk(std::false_type());
  }
  if (j >= a.T) return;
  const float factor = w.is_dk ? a.scale : 1.f;
  if (w.split && j < a.sinks) {
    // [b, hk, tile, part, dk / dv, key, D]
    float* out = a.parts + ((((((int64_t)w.b * a.Hkv + w.hk) * a.sink_tiles + w.tile) * (a.nchunks + 1) + w.part) *
                                 2 + !w.is_dk) * a.sink_rows + (j - w.k0)) * a.D;
    store_columns<float, DP>(out, acc, factor, a.D);
  } else if (w.part == 0) {   // (the chunks behind the window concern the sinks alone)
    T* out = (T*)(w.is_dk ? a.dk : a.dv) + (((int64_t)w.b * a.T + j) * a.Hkv + w.hk) * a.D;
    store_columns<T, DP>(out, acc, j < w.len ? factor : 0.f, a.D);
  }
}

// Adds the partial results of the sinks in order: one thread per element.
template <typename T>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(const Args a, int64_t total) {
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t per_tile = (int64_t)a.sink_rows * a.D;
    const int64_t in_tile = e % per_tile, which = e / per_tile % 2, tile = e / per_tile / 2 % a.sink_tiles;
    const int64_t bh = e / per_tile / 2 / a.sink_tiles;
    const int64_t j = tile * kQueries + in_tile / a.D, b = bh / a.Hkv, hk = bh % a.Hkv;
    if (j >= a.sinks) continue;
    const float* p = a.parts + ((bh * a.sink_tiles + tile) * (a.nchunks + 1) * 2 + which) * per_tile + in_tile;
    float s = 0.f;
    if (j < length_of(a, (int)b)) {
#pragma unroll 8
      for (int c = 0; c <= a.nchunks; ++c) s += p[(int64_t)c * 2 * per_tile];
    }
    T* out = (T*)(which ? a.dv : a.dk);
    out[((b * a.T + j) * a.Hkv + hk) * a.D + in_tile % a.D] = (T)s;
  }
}

// ------------------------------------------------------------------------------- host side
// Workgroups of a launch: threads are counted in 32 bits, and dk and dv take up to six workgroups for
// one of the others.  A larger batch is run in parts, one after the other.
constexpr int64_t kMaxGroups = ((1ll << 32) - 1) / kThreads / 6;
int64_t batch_of_launch(const mn_attention* d) {
  const int64_t tiles = (d->T + kQueries - 1) / kQueries, most = kMaxGroups / (tiles * d->Hq);
  return d->B < most ? d->B : most;
}

int check(const mn_attention* d) {
  if (!d || d->B < 0 || d->T < 0 || d->Hq <= 0 || d->Hkv <= 0 || d->D <= 0) return MN_EINVAL;
  if (d->Hq % d->Hkv || d->left < -1 || d->right < -1 || d->sinks < 0) return MN_EINVAL;
  if (!(d->scale > 0.f) || d->scale > 1e30f) return MN_EINVAL;
  if (d->D > kMaxD || d->T >= (1 << 28)) return MN_EUNSUPPORTED;
  const int64_t tiles = (d->T + kQueries - 1) / kQueries;
  if (d->B >= (1 << 28) || d->Hq >= (1 << 20)) return MN_EUNSUPPORTED;
  if (tiles && (d->Hq > kMaxGroups / tiles || d->B * d->Hq > (1ll << 28) / tiles)) return MN_EUNSUPPORTED;
  return MN_OK;
}

// "No limit" and limits beyond the sequence are T: sums with them stay inside 32 bits.
int32_t limit(int64_t v, int64_t T) { return (int32_t)(v < 0 || v > T ? T : v); }

// How the queries behind the window of the key tiles with sinks are cut: chunks that make 1024
// rows to walk over (all heads of the group), longer ones where that would be more than 128
// chunks, or more than two for each plain tile.  Shorter ones start and end more often than they
// multiply (T = 15808, four batches of 16 heads: 2.70 ms in chunks of 128, 2.32 of 1024), much
// longer ones outlast a plain tile.  Not cut where the sinks are more than an eighth of the keys
// (enough workgroups share the walk then).
void split_for(const mn_attention* d, Args* a) {
  a->sink_tiles = a->nchunks = 0;
  a->chunk = 1;
  const int64_t T = d->T, left = limit(d->left, T), all = (T + kQueries - 1) / kQueries;
  const int64_t sinks = d->sinks < T ? d->sinks : T, tiles = (sinks + kQueries - 1) / kQueries;
  const int64_t behind = T - kQueries - left;   // queries behind the window of the first tile
  if (sinks == 0 || behind <= 0 || tiles * kQueries * 8 > T) return;
  int64_t most = 2 * all / tiles;               // at least 16
  if (most > 128) most = 128;
  int64_t chunk = (behind + most - 1) / most;
  const int64_t rows = 1024 / (d->Hq / d->Hkv);
  chunk = chunk < rows ? rows : chunk;
  chunk = (chunk + 63) / 64 * 64;
  a->sink_tiles = (int32_t)tiles;
  a->sink_rows = (int32_t)(sinks < kQueries ? sinks : kQueries);
  a->chunk = (int32_t)chunk;
  a->nchunks = (int32_t)((behind + chunk - 1) / chunk);
}

size_t parts_floats(const mn_attention* d, const Args& a) {
  return (size_t)d->B * d->Hkv * a.sink_tiles * (a.nchunks + 1) * 2 * a.sink_rows * d->D;
}

Args args_for(const mn_attention* d) {
  Args a = {};
  for (int k = 0; k < 3; ++k) {
    a.sq[k] = d->q_stride[k];
    a.sk[k] = d->k_stride[k];
    a.sv[k] = d->v_stride[k];
  }
  a.T = (int32_t)d->T; a.Hq = d->Hq; a.Hkv = d->Hkv; a.D = d->D;
  a.left = limit(d->left, d->T); a.right = limit(d->right, d->T);
  a.sinks = (int32_t)(d->sinks < d->T ? d->sinks : d->T);
  a.tiles = (int32_t)((d->T + kQueries - 1) / kQueries);
  a.group = d->Hq / d->Hkv;
  a.fold = a.left != a.right && (a.left > a.T / 4 || a.right > a.T / 4);
  a.scale = d->scale;
  a.scale_log2 = d->scale * kLog2e;
  return a;
}

// f(head size rounded up to 32, can rows be loaded straight to LDS) as constants
template <int V, bool B>
struct Int {
  static constexpr int value = V;
  static constexpr bool direct = B;
};
template <typename F>
int for_width(int D, bool direct, F f) {
  if (D <= 32) return direct ? f(Int<32, true>()) : f(Int<32, false>());
  if (D <= 64) return direct ? f(Int<64, true>()) : f(Int<64, false>());
  if (D <= 96) return direct ? f(Int<96, true>()) : f(Int<96, false>());
  return direct ? f(Int<128, true>()) : f(Int<128, false>());
}

// f(the operator on a part of the batch, the part's first entry) until the batch is through.
template <typename F>
int in_parts(const mn_attention* desc, F f) {
  mn_attention d = *desc;
  const int64_t part = batch_of_launch(desc);
  for (int64_t b0 = 0; b0 < desc->B; b0 += part) {
    d.B = desc->B - b0 < part ? desc->B - b0 : part;
    const int st = f(&d, b0);
    if (st != MN_OK) return st;
  }
  return MN_OK;
}

// Loads straight to LDS move 16-byte chunks: rows have to start on 16 bytes and be whole chunks.
bool direct_rows(const void* p, const int64_t* stride, const mn_attention* d, int bytes) {
  const int64_t n = 16 / bytes;
  return mn_aligned(p, 16) && d->D % n == 0 && (d->B == 1 || stride[0] % n == 0) && stride[1] % n == 0 &&
         stride[2] % n == 0 && stride[1] >= 0 && stride[1] < (1 << 22);   // 64 rows in 31 bits
}

template <typename T, int DP>
constexpr int kLdsQ = 4 * Tile<T, DP, kRows<T>>::BYTES;   // two buffers of two tiles
template <typename T, int DP>
constexpr int kLdsKv = kLdsQ<T, DP> + 4 * kRows<T> * (int)sizeof(float);   // and two rows' statistics

// Dynamic LDS of more than 64 KB (dk / dv at D > 64) has to be asked for.
template <typename T, int DP, bool DIRECT>
bool raise_lds() {
  static_assert(kLdsQ<T, DP> <= 65536, "only dk / dv need more");
  return kLdsKv<T, DP> <= 65536 ||
         hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_dkv_kernel<T, DP, DIRECT>),
                             hipFuncAttributeMaxDynamicSharedMemorySize, kLdsKv<T, DP>) == hipSuccess;
}
template <typename T>
bool raise_lds_of() {
  return raise_lds<T, 64, false>() && raise_lds<T, 96, false>() && raise_lds<T, 128, false>() &&
         raise_lds<T, 64, true>() && raise_lds<T, 96, true>() && raise_lds<T, 128, true>();
}

}  // namespace

// Once per device: from mn_init, or from the first backward pass of a caller that never calls it.
bool mn_attention_init() {
  static std::mutex lock;
  static bool done[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
  std::lock_guard<std::mutex> hold(lock);
  if (!done[dev]) done[dev] = raise_lds_of<float>() && raise_lds_of<bf16_t>() && raise_lds_of<f16_t>();
  return done[dev];
}

extern "C" {

int mn_attention_fwd(const mn_attention* desc, const void* q, const void* k, const void* v, const int32_t* lengths,
                     void* out, float* lse, int dtype, mn_stream_t stream) {
  const int st = check(desc);
  if (st != MN_OK) return st;
  return mn_for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (desc->B == 0 || desc->T == 0) return (int)MN_OK;
    if (!q || !k || !v || !out || !lse) return (int)MN_EINVAL;
    return in_parts(desc, [&](const mn_attention* d, int64_t b0) {
      Args a = args_for(d);
      const int64_t tokens = b0 * d->T * d->Hq;
      a.q = (const T*)q + b0 * a.sq[0]; a.k = (const T*)k + b0 * a.sk[0]; a.v = (const T*)v + b0 * a.sv[0];
      a.o = (T*)out + tokens * d->D; a.lse = lse + tokens; a.lengths = lengths ? lengths + b0 : nullptr;
      const unsigned grid = (unsigned)(a.tiles * d->Hq * d->B);
      const bool direct = direct_rows(a.k, a.sk, desc, sizeof(T)) && direct_rows(a.v, a.sv, desc, sizeof(T));
      return for_width(d->D, direct, [&](auto w) {
        constexpr int DP = decltype(w)::value, lds = kLdsQ<T, DP>;
        constexpr bool DIRECT = decltype(w)::direct;
        attn_fwd_kernel<T, DP, DIRECT><<<grid, kThreads, lds, mn_stream(stream)>>>(a);
        return mn_launch_status();
      });
    });
  });
}

size_t mn_attention_bwd_ws_bytes(const mn_attention* desc) {
  if (check(desc) != MN_OK || desc->T == 0) return 0;
  mn_attention d = *desc;
  d.B = batch_of_launch(desc);   // (parts of the batch take turns with it)
  Args a = {};
  split_for(&d, &a);
  return ((size_t)d.B * d.Hq * d.T + parts_floats(&d, a)) * sizeof(float);
}

int mn_attention_bwd(const mn_attention* desc, const void* grad, const void* q, const void* k, const void* v,
                     const void* out, const float* lse, const int32_t* lengths, void* dq, void* dk, void* dv,
                     int dtype, void* ws, size_t ws_bytes, mn_stream_t stream) {
  const int st = check(desc);
  if (st != MN_OK) return st;
  return mn_for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (desc->B == 0 || desc->T == 0) return (int)MN_OK;
    if (!grad || !q || !k || !v || !out || !lse || !dq || !dk || !dv) return (int)MN_EINVAL;
    if (!ws || ws_bytes < mn_attention_bwd_ws_bytes(desc) || !mn_aligned(ws, 4)) return (int)MN_EINVAL;
    return in_parts(desc, [&](const mn_attention* d, int64_t b0) {
      Args a = args_for(d);
      const int64_t tokens = b0 * d->T * d->Hq, key_tokens = b0 * d->T * d->Hkv;
      a.q = (const T*)q + b0 * a.sq[0]; a.k = (const T*)k + b0 * a.sk[0]; a.v = (const T*)v + b0 * a.sv[0];
      a.out = (const T*)out + tokens * d->D; a.grad = (const T*)grad + tokens * d->D;
      a.lse = const_cast<float*>(lse) + tokens; a.dq = (T*)dq + tokens * d->D;
      a.dk = (T*)dk + key_tokens * d->D; a.dv = (T*)dv + key_tokens * d->D;
      a.lengths = lengths ? lengths + b0 : nullptr;
      a.delta = (float*)ws;
      a.parts = a.delta + (size_t)d->B * d->Hq * d->T;
      split_for(d, &a);
      hipStream_t s = mn_stream(stream);
      const bool direct = direct_rows(a.k, a.sk, desc, sizeof(T)) && direct_rows(a.v, a.sv, desc, sizeof(T)) &&
                          direct_rows(a.q, a.sq, desc, sizeof(T)) && mn_aligned(grad, 16) &&
                          (int64_t)d->Hq * d->D < (1 << 22);
      const int rc = for_width(d->D, direct, [&](auto w) {
        constexpr bool DIRECT = decltype(w)::direct;
        constexpr int DP = decltype(w)::value, lds_q = kLdsQ<T, DP>, lds_kv = kLdsKv<T, DP>;
        if (lds_kv > 65536 && !mn_attention_init()) return (int)MN_ELAUNCH;
        attn_dq_kernel<T, DP, DIRECT><<<(unsigned)(a.tiles * d->Hq * d->B), kThreads, lds_q, s>>>(a);
        const unsigned items = (unsigned)(a.tiles + a.sink_tiles * a.nchunks);
        attn_dkv_kernel<T, DP, DIRECT><<<(unsigned)(2 * items * d->Hkv * d->B), kThreads, lds_kv, s>>>(a);
        return mn_launch_status();
      });
      if (rc != MN_OK || !a.sink_tiles) return rc;
      const int64_t total = d->B * d->Hkv * a.sink_tiles * 2 * a.sink_rows * d->D;
      const int64_t groups = (total + kThreads - 1) / kThreads;
      attn_join_kernel<T><<<(unsigned)(groups < (1 << 20) ? groups : 1 << 20), kThreads, 0, s>>>(a, total);
      return mn_launch_status();
    });
  });
}

}  // extern "C"
