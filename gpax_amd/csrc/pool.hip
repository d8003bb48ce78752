// pool.hip — a pool of candidates over time: the weight each candidate gathers from the rows of a policy (posterior draws),
// and the eviction that keeps a pool within its budget by that weight.
//
// weights: w'_j = decay w_j + sum over rows of u_r p_rj.  Bound by memory: a score is read once where a row fits a workgroup's
// registers (16 candidates per lane, up to 16384), twice beyond that.  Every lane owns its candidates for all rows that its
// team works off, so the sums stay in registers; the partial sums of the teams are added in a fixed order, without atomics:
// the same bits every time.
//
// eviction: of a pool's `length` candidates the first, the most recent and those of largest weight stay, in their order.
#include "pool.h"

using namespace gpx;

namespace {

struct WeightArgs {
  PoolScores sc;
  const void* row_weights; // pools x R contiguous, or nullptr
  const void* weights;     // pools x M contiguous, or nullptr: zeros
  void* out;               // pools x M
  void* part;              // pools x groups x M partial sums when groups > 1
  const void* stats;       // column pass: rows x {m, log2 s}, or, where a row has several splits, ...
  const void* parts;       // ... rows x splits partial results (choice.hip)
  int splits;
  double decay;
  int groups;
};

constexpr int PER_LANE = 16; // candidates a lane owns in the one-pass kernel
constexpr int TEAMS = 8;     // rows at a time of a workgroup in which a row is a wave's
// the most waves for a row: 16 sums and 16 scores of 64 bits do not fit the 128 registers that 16 waves leave each lane
inline int team_waves(int dtype) { return dtype == GPX_DTYPE_F64 ? 8 : 16; }

// finished sums of candidates j .. j + VEC, of them those from `from` on: straight to the output, or to this group's partial sums
template <typename A, int VEC>
__device__ __forceinline__ void store_sums(const WeightArgs& a, int64_t b, int group, int64_t from, int64_t j, const A* acc) {
  const int64_t M = a.sc.M;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (j + e < from) continue;
    if (j + e >= M) return;
    if (a.groups > 1) {
      static_cast<A*>(a.part)[(b * a.groups + group) * M + j + e] = acc[e];
    } else {
      const A old = a.weights ? (A)a.decay * static_cast<const A*>(a.weights)[b * M + j + e] : (A)0;
      static_cast<A*>(a.out)[b * M + j + e] = old + acc[e];
    }
  }
}

// One pass over pools of at most 1024 candidates: a row a wave, TEAMS waves per workgroup, no barrier before the end.  Bound by
// the latency of a row or two per wave: 1000 x 1024 float64 take 8.5 us and 4.7 to join (8.2 MB, 1 TB/s), 4000 x 1024 float32
// 7.2 and 8.4; four waves a row take 13.1 and 6.3, 16.2 and 13.4.
template <typename T>
__global__ __launch_bounds__(TEAMS * 64) void pool_weights_wave_kernel(WeightArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value, U = PER_LANE / VEC, SPAN = 64 * VEC;
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t b = blockIdx.y;
  A acc[PER_LANE];
#pragma unroll
  for (int e = 0; e < PER_LANE; ++e) acc[e] = (A)0;
  for (int64_t r = (int64_t)blockIdx.x * TEAMS + team; r < a.sc.R; r += (int64_t)a.groups * TEAMS) {
    const A u = a.row_weights ? static_cast<const A*>(a.row_weights)[b * a.sc.R + r] : (A)1;
    if (u == (A)0) continue; // uniform
    const A c = temperature_scale(row_temperature<A>(a.sc, b, r));
    const Row<T> v = row_view<T>(a.sc, b, r);
    A x[PER_LANE];
    load_step<T, VEC, U>(v, 0, SPAN, lane * VEC, x);
    const int live = (v.n + SPAN - 1) / (SPAN); // vectors of the lanes that the row reaches into
    A m = x[0];
#pragma unroll
    for (int e = 1; e < PER_LANE; ++e) m = fmax(m, x[e]);
    m = wave_max(m);
    const A ref = finite_max(m);
    A s = (A)0;
#pragma unroll
    for (int w = 0; w < U; ++w) {
      if (w >= live) break; // uniform
#pragma unroll
      for (int e = w * VEC; e < (w + 1) * VEC; ++e) {
        x[e] = exp2_acc((x[e] - ref) * c);
        s += x[e];
      }
    }
    s = wave_sum(s);
    if (s == (A)0) continue; // nothing in this row may be chosen
    const A f = u / s;
    if (!(fabs(f) < (A)INFINITY)) { // infinite or NaN for what may be chosen, nothing for what may not (0 f would be NaN)
      load_step<T, VEC, U>(v, 0, SPAN, lane * VEC, x);
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) acc[e] += x[e] == neg_inf<A>() ? (A)0 : exp2_acc((x[e] - ref) * c) * f;
    } else {
#pragma unroll
      for (int w = 0; w < U; ++w) {
        if (w >= live) break;
#pragma unroll
        for (int e = w * VEC; e < (w + 1) * VEC; ++e) acc[e] = fma(x[e], f, acc[e]);
      }
    }
  }
  // the waves' sums in their order, into the first one's registers
  __shared__ A sum[64 * PER_LANE];
  for (int t = TEAMS - 1; t > 0; --t) {
    if (team == t) {
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) sum[e * 64 + lane] = (t == TEAMS - 1 ? (A)0 : sum[e * 64 + lane]) + acc[e];
    }
    __syncthreads();
  }
  if (team != 0) return;
#pragma unroll
  for (int e = 0; e < PER_LANE; ++e) acc[e] += sum[e * 64 + lane];
#pragma unroll
  for (int w = 0; w < U; ++w) store_sums<A, VEC>(a, b, blockIdx.x, 0, w * SPAN + lane * VEC, acc + w * VEC);
}

// One pass over longer pools: a row a workgroup of WAVES waves, which meet at a barrier for the largest score and at one for the
// sum.  What is needed of the rows (scale, weight, length) is fetched for 64 at a time, and the next row's scores are on their
// way while one is worked on (DENSE: candidates, and mask bytes, side by side; else they are loaded where they are used).
// One workgroup of 16 waves fills a CU's registers, so a row's two barriers and reductions stand in the open: 2048 x 16384
// float32 take 33.5 us (4.0 TB/s; 20 vector instructions a score occupy the vector units for 55 % of it; of its registers, 128 at
// most, 3 spill), 16 x 128 x 16381 35 us, with rows half as long on average 32, and 7 to join.  The two passes of longer pools
// would take 51 and 52.  4 waves up to 4096 candidates: 2000 x 4096 float32 12.6 us and 8.6 to join, with 16 waves 21.5 and 4.6;
// float64 1000 x 4096 17.3 against 19.6.
constexpr int ROW_BLOCK = 64;
template <typename A>
struct WorkRow {
  A c, u;
  int n;
};
template <typename T, int WAVES, bool DENSE>
__global__ __launch_bounds__(WAVES * 64) void pool_weights_kernel(WeightArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value, U = PER_LANE / VEC, LANES = WAVES * 64, SPAN = LANES * VEC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = threadIdx.x, M = a.sc.M;
  const int64_t b = blockIdx.y;
  __shared__ WorkRow<A> rows[ROW_BLOCK];
  __shared__ A red[2][WAVES]; // each half is read before the barrier of the other one, and written after it
  A acc[PER_LANE];
#pragma unroll
  for (int e = 0; e < PER_LANE; ++e) acc[e] = (A)0;
  const int64_t stride = a.groups;
  RawStep<T, VEC, U, DENSE> raw;
  const T* x0 = static_cast<const T*>(a.sc.x) + b * a.sc.xb;
  const uint8_t* mask0 = a.sc.mask ? a.sc.mask + b * a.sc.mb : nullptr;
#pragma unroll 1
  for (int64_t r0 = blockIdx.x; r0 < a.sc.R; r0 += stride * ROW_BLOCK) {
    const int64_t left = (a.sc.R - r0 + stride - 1) / stride;
    const int count = left < ROW_BLOCK ? (int)left : ROW_BLOCK;
    __syncthreads();
    if (at < count) {
      const int64_t r = r0 + at * stride;
      WorkRow<A> k;
      k.u = a.row_weights ? static_cast<const A*>(a.row_weights)[b * a.sc.R + r] : (A)1;
      k.c = temperature_scale(row_temperature<A>(a.sc, b, r));
      k.n = k.u == (A)0 ? 0 : row_length(a.sc, b, r);
      rows[at] = k;
    }
    __syncthreads();
    auto row = [&](int q) {
      WorkRow<A> k = rows[q];
      k.n = __builtin_amdgcn_readfirstlane(k.n);
      return k;
    };
    auto view = [&](int q, int n) {
      const int64_t r = r0 + q * stride;
      return Row<T>{x0 + r * a.sc.xr, mask0 ? mask0 + r * a.sc.mr : nullptr, a.sc.xc, a.sc.mc, n};
    };
    WorkRow<A> next = row(0);
    if (DENSE) raw.load(view(0, next.n), M, SPAN, at * VEC);
#pragma unroll 1
    for (int q = 0; q < count; ++q) {
      const WorkRow<A> k = next;
      A x[PER_LANE];
      if (DENSE) raw.decode(mask0 != nullptr, k.n, M, SPAN, at * VEC, x);
      if (q + 1 < count) {
        next = row(q + 1);
        if (DENSE) raw.load(view(q + 1, next.n), M, SPAN, at * VEC);
      }
      if (k.n == 0) continue;
      if (!DENSE) load_step<T, VEC, U>(view(q, k.n), 0, SPAN, at * VEC, x);
      const A c = k.c, u = k.u;
      const int n = k.n;
      A m = x[0];
#pragma unroll
      for (int e = 1; e < PER_LANE; ++e) m = fmax(m, x[e]);
      m = wave_max(m);
      if ((threadIdx.x & 63) == 0) red[0][wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmax(m, red[0][w]);
      const A ref = finite_max(m);
      A s = (A)0;
      uint32_t there = 0; // which of this lane's candidates exist, for a row that is not finite
#pragma unroll
      for (int w = 0; w < U; ++w) {
        if (w * SPAN >= n) break; // uniform
#pragma unroll
        for (int e = w * VEC; e < (w + 1) * VEC; ++e) {
          there |= (uint32_t)(x[e] != neg_inf<A>()) << e;
          x[e] = exp2_acc((x[e] - ref) * c);
          s += x[e];
        }
      }
      s = wave_sum(s);
      if ((threadIdx.x & 63) == 0) red[1][wave] = s;
      __syncthreads();
      s = (A)0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += red[1][w];
      if (s == (A)0) continue; // nothing in this row may be chosen
      const A f = u / s;
      if (!(fabs(f) < (A)INFINITY)) { // infinite or NaN for what may be chosen, nothing for what may not (0 f would be NaN)
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) acc[e] += (there >> e) & 1 ? x[e] * f : (A)0;
      } else {
#pragma unroll
        for (int w = 0; w < U; ++w) {
          if (w * SPAN >= n) break;
#pragma unroll
          for (int e = w * VEC; e < (w + 1) * VEC; ++e) acc[e] = fma(x[e], f, acc[e]);
        }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < U; ++w) {
    const int j = w * SPAN + at * VEC;
    store_sums<A, VEC>(a, b, blockIdx.x, j, DENSE && j > M - VEC ? M - VEC : j, acc + w * VEC);
  }
}

// Second pass over longer pools: a workgroup sums a tile of 256 lanes' vectors over its share of rows.  What it needs of a row
// (scale, reference, log of the sum, weight, length) it joins itself from the first pass's partial results, 64 rows at a time in
// LDS; the next row that reaches into the tile is on its way while one is worked on; a mask that all rows share is read once.
// A vector that would cross the end of the pool starts earlier, and only its own candidates are written.  DENSE: candidates (and
// mask bytes) side by side.  64 x 262144 float64 with a shared mask: 36 us (3.7 TB/s, behind 28 us of the first pass), float32
// 15.6 us (4.3 TB/s), bfloat16 16.2: exponentials and 64-bit arithmetic (60 vector instructions a score in float64, which occupy
// the vector units for 72 % of the time), then memory.
constexpr int COL_BLOCK = 64;
constexpr int col_vecs(int size) { return size == 2 ? 1 : 2; } // vectors a lane holds of a row (one is 8 scores of 16 bits)
template <typename A>
struct ColumnRow {
  A c, m, log2s, u;
  int n;
};
template <typename T, bool DENSE>
__global__ __launch_bounds__(256) void pool_columns_kernel(WeightArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value, SPAN = 256 * VEC, U = col_vecs(sizeof(T)), E = VEC * U;
  __shared__ ColumnRow<A> rows[COL_BLOCK];
  const int64_t b = blockIdx.z;
  const int M = a.sc.M, j0 = (int)blockIdx.x * SPAN * U;
  const int64_t per = (a.sc.R + a.groups - 1) / a.groups;
  const int64_t r0 = per * blockIdx.y, r1 = r0 + per < a.sc.R ? r0 + per : a.sc.R;
  A acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = (A)0;
  int off[U]; // this lane's vectors; a pool that comes here has more than a vector's candidates
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int start = j0 + u * SPAN + (int)threadIdx.x * VEC;
    off[u] = start < M - VEC ? start : M - VEC;
  }
  const T* x = static_cast<const T*>(a.sc.x) + b * a.sc.xb;
  const uint8_t* mask = a.sc.mask ? a.sc.mask + b * a.sc.mb : nullptr;
  Pack<T, VEC> next[U];
  MaskPack<VEC> next_mask[U];
  auto load_mask = [&](const uint8_t* m) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (DENSE) {
        next_mask[u] = *reinterpret_cast<const MaskPack<VEC>*>(m + (uint32_t)off[u]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) next_mask[u].v[e] = m[(off[u] + e) * a.sc.mc];
      }
    }
  };
  auto load = [&](int64_t r) {
    const T* row = x + r * a.sc.xr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (DENSE) {
        next[u] = *reinterpret_cast<const Pack<T, VEC>*>(row + (uint32_t)off[u]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) next[u].v[e] = row[(off[u] + e) * a.sc.xc];
      }
    }
    if (mask && a.sc.mr != 0) load_mask(mask + r * a.sc.mr);
  };
  if (mask && a.sc.mr == 0) load_mask(mask);
#pragma unroll 1
  for (int64_t block = r0; block < r1; block += COL_BLOCK) {
    __syncthreads();
    // 16 lanes a row, a partial result each
    const int count = (int)(r1 - block < COL_BLOCK ? r1 - block : COL_BLOCK);
#pragma unroll 1
    for (int i = 0; i * 16 < count; ++i) {
      const int local = i * 16 + ((int)threadIdx.x >> 4);
      const int64_t r = block + local < r1 ? block + local : r1 - 1, row = b * a.sc.R + r;
      ColumnRow<A> k;
      k.c = temperature_scale(row_temperature<A>(a.sc, b, r));
      k.u = a.row_weights ? static_cast<const A*>(a.row_weights)[row] : (A)1;
      k.n = row_length(a.sc, b, r);
      row_reference(a.stats, a.parts, a.splits, row, k.c, (int)threadIdx.x & 15, k.m, k.log2s);
      if (k.u == (A)0 || k.m == neg_inf<A>()) k.n = 0; // weight 0, or nothing that may be chosen (and no NaN: that has no largest)
      if (k.u != (A)0 && k.log2s != k.log2s) k.n = row_length(a.sc, b, r);
      if ((threadIdx.x & 15) == 0) rows[local] = k;
    }
    __syncthreads();
    ColumnRow<A> k = rows[0], kn = k;
    if (j0 < k.n) load(block); // uniform: the row reaches into the tile
#pragma unroll 1
    for (int q = 0; q < count; ++q, k = kn) {
      kn = rows[q + 1 < count ? q + 1 : q];
      Pack<T, VEC> p[U];
      MaskPack<VEC> ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        p[u] = next[u];
        ok[u] = next_mask[u];
      }
      if (q + 1 < count && j0 < kn.n) load(block + q + 1);
      if (j0 >= k.n) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const A v = to_acc(p[e / VEC].v[e % VEC]);
        const A w = k.u * exp2_acc((v - k.m) * k.c - k.log2s);
        const bool in = off[e / VEC] + e % VEC < k.n && (!mask || ok[e / VEC].v[e % VEC]) && v != neg_inf<A>();
        acc[e] += in ? w : (A)0;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) store_sums<A, VEC>(a, b, blockIdx.y, j0 + u * SPAN + (int)threadIdx.x * VEC, off[u], acc + u * VEC);
}

// decay w + the groups' partial sums in their order: 64 candidates per workgroup, the groups dealt to its four waves.  4 to 9 us,
// most of it the launch (16 x 16 groups x 16381: 17 MB, 6 us).
template <typename A>
__global__ __launch_bounds__(256) void pool_weights_join_kernel(WeightArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t M = a.sc.M, b = blockIdx.y, j = (int64_t)blockIdx.x * 64 + lane;
  __shared__ A sh[4][64];
  A s = (A)0;
  if (j < M) {
    const int per = (a.groups + 3) / 4;
    const int g1 = per * (wave + 1) < a.groups ? per * (wave + 1) : a.groups;
    const A* p = static_cast<const A*>(a.part) + b * a.groups * M + j;
#pragma unroll 8
    for (int g = per * wave; g < g1; ++g) s += p[(int64_t)g * M];
  }
  sh[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < M) {
    const A old = a.weights ? (A)a.decay * static_cast<const A*>(a.weights)[b * M + j] : (A)0;
    static_cast<A*>(a.out)[b * M + j] = old + (((sh[0][lane] + sh[1][lane]) + sh[2][lane]) + sh[3][lane]);
  }
}

// ---- eviction ---------------------------------------------------------------------------------------------------------
//
// What stays of a pool of L > budget candidates: the `first` first, the `recent` last, and of the others the `need` of largest
// weight.  The need-th largest is found on integers of the weights' order, digit by digit from the highest bit in which they
// differ at all, by histograms; a digit that holds exactly what is still needed ends the search.  Candidates above the found
// prefix stay, of those equal to it the first in order.  Counts only: no result depends on the order of an atomic.
//
// One workgroup per pool where the pool fits its registers (16384 candidates).  Longer pools are cut into chunks of 4096, a
// workgroup each, over six launches: range of the keys | histograms of 12, 12 and 12 bits | the few candidates that share all
// 36 (or that need no telling apart) | output.  Read six times, but 2 MB of weights stay in the caches: bound by the launches.
// 64-bit weights of many or very long pools (REREADS_MAX) have a histogram for every 12 bits of a key.

constexpr int EVICT_PAYLOADS = 16;
// Payload rows up to this are moved by the lane that keeps the candidate, longer ones by a launch of their own: of 64 pools of
// 16384, cut to 4096, rows of 24 bytes take 26.6 us in all against 20.9 + 4.5, of 64 bytes 36.9 against 22.0 + 7.9.
constexpr int FUSED_ROW_BYTES = 32;

struct Payload {
  const char* src;
  char* dst;
  int bytes, unit; // of a row; of one access
};
struct EvictArgs {
  const void* weights; // pools x M
  const void* lengths;
  int len64;
  int64_t ls; // stride of lengths
  int64_t M, K, first, recent;
  int64_t* indices; // pools x K
  int64_t* new_lengths;
  void* out; // pools x K
  int npay;
  void* ws;
  int64_t chunks;
  int levels; // histograms
  Payload pay[EVICT_PAYLOADS];
};

// weights as integers of the same order; NaN lowest, -0 = +0
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double w) {
  if (w != w) return 0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(w + 0.0);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
template <typename W>
struct KeyOf {
  typedef uint32_t type;
};
template <>
struct KeyOf<double> {
  typedef uint64_t type;
};
// key >> shift where shift may be all of the key's bits
template <typename Key>
__device__ __forceinline__ Key above(Key k, int shift) {
  return shift >= (int)sizeof(Key) * 8 ? (Key)0 : k >> (shift & (int)(sizeof(Key) * 8 - 1));
}
template <typename Key>
__device__ __forceinline__ int bits_of(Key diff) {
  return diff == 0 ? 0 : (int)sizeof(Key) * 8 - (sizeof(Key) == 8 ? __clzll((long long)diff) : __clz((int)diff));
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* sh, F f) { // 16 waves; sh: 16 values, not reused before the next barrier
  v = wave_reduce(v, f);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < 16; ++i) v = f(v, sh[i]);
  return v;
}
template <typename Key>
__device__ __forceinline__ Key key_and(Key x, Key y) {
  return x & y;
}
template <typename Key>
__device__ __forceinline__ Key key_or(Key x, Key y) {
  return x | y;
}

struct PoolCut { // what a pool's length leaves to decide
  int64_t L, keep, lo, hi; // candidates lo .. hi - 1 are free to go
  uint32_t need;           // how many of them stay
};
__device__ __forceinline__ PoolCut pool_cut(const EvictArgs& a, int64_t b) {
  PoolCut c;
  c.L = a.M;
  if (a.lengths) {
    c.L = a.len64 ? static_cast<const int64_t*>(a.lengths)[b * a.ls] : (int64_t)static_cast<const int32_t*>(a.lengths)[b * a.ls];
    c.L = c.L < 0 ? 0 : (c.L > a.M ? a.M : c.L);
  }
  const bool all = c.L <= a.K;
  c.keep = all ? c.L : a.K;
  c.lo = all ? 0 : a.first;
  c.hi = all ? 0 : c.L - a.recent;
  c.need = all ? 0u : (uint32_t)(a.K - a.first - a.recent);
  return c;
}

struct Digit { // where the need-th largest lies in a histogram, counted from the top
  int bin;
  uint32_t above, count;
};
constexpr int WIDE_BITS = 12, WIDE_BINS = 1 << WIDE_BITS;
// The 12-bit digit that the need-th largest lies in: four bins a lane, sums from the top by wave and over the waves
__device__ __forceinline__ Digit wide_digit(const uint32_t* hist, uint32_t need) {
  static_assert(WIDE_BINS == 4 * 1024, "four bins a lane");
  __shared__ uint32_t totals[16];
  __shared__ Digit found;
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t c[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * tid + i];
  uint32_t upto = sum; // of this lane and all above it in the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t v = __shfl_down(upto, o);
    if (lane + o < 64) upto += v;
  }
  if (lane == 0) totals[tid >> 6] = upto;
  __syncthreads();
  for (int w = (tid >> 6) + 1; w < 16; ++w) upto += totals[w];
  uint32_t over = upto - sum;
  if (over < need && need <= upto) { // one lane of the workgroup
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      if (over < need && need <= over + c[i]) found = Digit{4 * tid + i, over, c[i]};
      over += c[i];
    }
  }
  __syncthreads();
  return found;
}

typedef uint32_t Unit16 __attribute__((ext_vector_type(4)));
constexpr int PUT = 4; // candidates a lane moves at a time: their loads are in flight together
// (Those past the end move the first one's row, and do not store it.)  N units of every row in flight.
template <typename Unit, int N>
__device__ __forceinline__ void move_part(Unit* dst, const Unit* s0, const Unit* s1, const Unit* s2, const Unit* s3, int n, int64_t step) {
  Unit u0[N], u1[N], u2[N], u3[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u0[i] = s0[i];
    u1[i] = s1[i];
    u2[i] = s2[i];
    u3[i] = s3[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    dst[i] = u0[i];
    if (n > 1) dst[step + i] = u1[i];
    if (n > 2) dst[2 * step + i] = u2[i];
    if (n > 3) dst[3 * step + i] = u3[i];
  }
}
template <typename Unit>
__device__ __forceinline__ void move_rows(char* dst, const char* s0, const char* s1, const char* s2, const char* s3, int n, int bytes) {
  Unit* d = reinterpret_cast<Unit*>(dst);
  const Unit *r0 = reinterpret_cast<const Unit*>(s0), *r1 = reinterpret_cast<const Unit*>(s1);
  const Unit *r2 = reinterpret_cast<const Unit*>(s2), *r3 = reinterpret_cast<const Unit*>(s3);
  const int units = bytes / (int)sizeof(Unit);
  const int64_t step = (int64_t)1024 * units;
  int i = 0;
  for (; i + 4 <= units; i += 4) move_part<Unit, 4>(d + i, r0 + i, r1 + i, r2 + i, r3 + i, n, step);
  switch (units - i) { // uniform
    case 3: move_part<Unit, 3>(d + i, r0 + i, r1 + i, r2 + i, r3 + i, n, step); break;
    case 2: move_part<Unit, 2>(d + i, r0 + i, r1 + i, r2 + i, r3 + i, n, step); break;
    case 1: move_part<Unit, 1>(d + i, r0 + i, r1 + i, r2 + i, r3 + i, n, step); break;
    default: break;
  }
}
// candidates j0 + kept[0 .. count) of pool b become those that stay from place pos0 on
template <typename W>
__device__ __forceinline__ void put_kept(const EvictArgs& a, int64_t b, int64_t pos0, int64_t j0, const uint16_t* kept, int count) {
  constexpr int T = 1024; // threads
  for (int p0 = threadIdx.x; p0 < count; p0 += PUT * T) {
    const int n = (count - p0 + T - 1) / T; // of this lane's, at most PUT are moved now
    const int64_t at = b * a.K + pos0 + p0;
    const int64_t j_0 = j0 + kept[p0], j_1 = n > 1 ? j0 + kept[p0 + T] : j_0;
    const int64_t j_2 = n > 2 ? j0 + kept[p0 + 2 * T] : j_0, j_3 = n > 3 ? j0 + kept[p0 + 3 * T] : j_0;
    const W* w = static_cast<const W*>(a.weights) + b * a.M;
    W* out = static_cast<W*>(a.out) + at;
    const W w0 = w[j_0], w1 = w[j_1], w2 = w[j_2], w3 = w[j_3];
    a.indices[at] = j_0;
    out[0] = w0;
    if (n > 1) a.indices[at + T] = j_1, out[T] = w1;
    if (n > 2) a.indices[at + 2 * T] = j_2, out[2 * T] = w2;
    if (n > 3) a.indices[at + 3 * T] = j_3, out[3 * T] = w3;
    for (int y = 0; y < a.npay; ++y) {
      const int64_t bytes = a.pay[y].bytes;
      const char* s = a.pay[y].src + b * a.M * bytes;
      const char *s0 = s + j_0 * bytes, *s1 = s + j_1 * bytes, *s2 = s + j_2 * bytes, *s3 = s + j_3 * bytes;
      char* d = a.pay[y].dst + at * bytes;
      switch (a.pay[y].unit) {
        case 16: move_rows<Unit16>(d, s0, s1, s2, s3, n, (int)bytes); break;
        case 8: move_rows<uint64_t>(d, s0, s1, s2, s3, n, (int)bytes); break;
        case 4: move_rows<uint32_t>(d, s0, s1, s2, s3, n, (int)bytes); break;
        default: move_rows<uint8_t>(d, s0, s1, s2, s3, n, (int)bytes); break;
      }
    }
  }
}
// places pos of pool b that nothing stays in
template <typename W>
__device__ __forceinline__ void put_nothing(const EvictArgs& a, int64_t b, int64_t pos) {
  const int64_t at = b * a.K + pos;
  a.indices[at] = -1;
  static_cast<W*>(a.out)[at] = (W)0;
  for (int y = 0; y < a.npay; ++y)
    for (int i = 0; i < a.pay[y].bytes; ++i) a.pay[y].dst[at * a.pay[y].bytes + i] = 0;
}

// Exclusive sums, in the order (i, wave), of the PER x 16 pairs of counts in LDS, from (g0, e0) on; by wave 0.
template <int PER>
__device__ __forceinline__ void exclusive_counts(uint32_t* cnt_g, uint32_t* cnt_e, uint32_t g0, uint32_t e0, int lane) {
  constexpr int N = (PER * 16 + 63) / 64;
  uint32_t g[N], e[N], sg = 0, se = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = N * lane + i < PER * 16;
    g[i] = sg;
    e[i] = se;
    sg += in ? cnt_g[N * lane + i] : 0;
    se += in ? cnt_e[N * lane + i] : 0;
  }
  uint32_t pg = sg, pe = se;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t vg = __shfl_up(pg, o), ve = __shfl_up(pe, o);
    if (lane >= o) {
      pg += vg;
      pe += ve;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (N * lane + i < PER * 16) {
      cnt_g[N * lane + i] = g0 + pg - sg + g[i];
      cnt_e[N * lane + i] = e0 + pe - se + e[i];
    }
}

// The candidates of 1024 PER places from j0 on, each lane's as bits g (stays), e (stays if among the first `need` of its
// kind): to their places, behind the g0 and e0 of the candidates before j0.  Compacted in LDS first, so that the outputs are
// written side by side.
template <typename W, int PER>
__device__ __forceinline__ void put_marked(const EvictArgs& a, int64_t b, int64_t j0, uint32_t g_bits, uint32_t e_bits, uint32_t need, uint32_t g0,
                                           uint32_t e0, int lane, int wave) {
  __shared__ uint32_t cnt_g[PER * 16], cnt_e[PER * 16];
  __shared__ uint16_t kept[PER * 1024];
  __shared__ int total;
#pragma unroll 1
  for (int i = 0; i < PER; ++i) {
    const uint64_t bg = __ballot((g_bits >> i) & 1), be = __ballot((e_bits >> i) & 1);
    if (lane == 0) {
      cnt_g[i * 16 + wave] = (uint32_t)__popcll(bg);
      cnt_e[i * 16 + wave] = (uint32_t)__popcll(be);
    }
  }
  __syncthreads();
  if (wave == 0) exclusive_counts<PER>(cnt_g, cnt_e, g0, e0, lane);
  __syncthreads();
  const uint32_t base = g0 + (e0 < need ? e0 : need);
#pragma unroll 1
  for (int i = 0; i < PER; ++i) {
    const bool g = (g_bits >> i) & 1, e = (e_bits >> i) & 1;
    const uint64_t bg = __ballot(g), be = __ballot(e), below = (1ull << lane) - 1;
    const uint32_t ng = cnt_g[i * 16 + wave] + (uint32_t)__popcll(bg & below);
    const uint32_t ne = cnt_e[i * 16 + wave] + (uint32_t)__popcll(be & below);
    const uint32_t at = ng + (ne < need ? ne : need) - base;
    const bool stays = g || (e && ne < need);
    if (stays) kept[at] = (uint16_t)(i * 1024 + threadIdx.x);
    if (i == PER - 1 && threadIdx.x == 1023) total = (int)(at + stays);
  }
  __syncthreads();
  put_kept<W>(a, b, base, j0, kept, total);
}

// One workgroup per pool of at most 1024 PER candidates, whose keys stay in its registers: a chain of barriers (range, two or three
// histograms of 12 bits, places), 9 us for 1000 candidates, 12 for 4096, 22 for 16384, 27 for 64 pools of that.  Over six
// launches 16384 take 32 us and the gaps between them, 64 pools of that 38.
template <typename W, int PER>
__global__ __launch_bounds__(1024) void pool_evict_kernel(EvictArgs a) {
  typedef typename KeyOf<W>::type Key;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t b = blockIdx.x;
  const W* w = static_cast<const W*>(a.weights) + b * a.M;
  const PoolCut cut = pool_cut(a, b);
  uint32_t need = cut.need;

  __shared__ uint32_t bins[WIDE_BINS];
  __shared__ Key sh_keys[2][16];

  Key key[PER];
  uint32_t free_bits = 0, g_bits = 0, e_bits = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t j = i * 1024 + tid;
    key[i] = j < cut.L ? order_key(w[j]) : (Key)0;
    const bool fr = j >= cut.lo && j < cut.hi;
    free_bits |= (uint32_t)fr << i;
    g_bits |= (uint32_t)(j < cut.L && !fr) << i;
  }
  if (need > 0) {
    Key all = ~(Key)0, any = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((free_bits >> i) & 1) {
        all &= key[i];
        any |= key[i];
      }
    all = block_reduce(all, sh_keys[0], key_and<Key>);
    any = block_reduce(any, sh_keys[1], key_or<Key>);
    int shift = bits_of<Key>(all ^ any);
    Key prefix = above(all, shift); // shift == 0: every weight is the same
    while (shift > 0) {
      const int lo = shift > WIDE_BITS ? shift - WIDE_BITS : 0, width = shift - lo;
      for (int i = tid; i < WIDE_BINS; i += 1024) bins[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (((free_bits >> i) & 1) && above(key[i], shift) == prefix) atomicAdd(&bins[(uint32_t)(key[i] >> lo) & ((1u << width) - 1u)], 1u);
      __syncthreads();
      const Digit d = wide_digit(bins, need);
      prefix = (prefix << width) | (Key)d.bin; // (a prefix of no bits is 0)
      need -= d.above;
      shift = lo;
      if (need == d.count) break; // the whole digit stays
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const Key hi = above(key[i], shift);
      const uint32_t fr = (free_bits >> i) & 1;
      g_bits |= (fr & (uint32_t)(hi > prefix)) << i;
      e_bits |= (fr & (uint32_t)(hi == prefix)) << i;
    }
  }
  put_marked<W, PER>(a, b, 0, g_bits, e_bits, need, 0, 0, lane, wave);
  for (int64_t p = cut.keep + tid; p < a.K; p += 1024) put_nothing<W>(a, b, p);
  if (tid == 0) a.new_lengths[b] = cut.keep;
}

// ---- longer pools: chunks of 4096, six launches and more ----
constexpr int CHUNK_PER = 4, CHUNK = 1024 * CHUNK_PER;
constexpr int MAX_TIED = 1024; // candidates told apart one by one in the last launch
// Three digits are all of a 32-bit key.  Of a 64-bit one they leave those that agree in 36 bits, counted from the highest that
// differs, to the last launch; if those are many, the workgroup of each chunk goes through all chunks of its pool.  (After two
// digits that already happens to weights within 2^-14 of each other beside one that is larger; the third launch costs 3 us.)  Up
// to this many chunks read by all workgroups together (one pool of 2^19 candidates, 64 of 65536) that is accepted; beyond it
// there is a launch for every digit that a key has.  Ordinary weights, and weights that all agree in 36 bits beside one that does
// not, with three digits and with six: 1 x 262144 35 and 240 us, 42 and 58; 1 x 524288 36 and 493, 43 and 61; 64 x 65536 93 and
// 470, 103 and 164; 64 x 131072 172 and 1546, 188 and 300; 64 x 524288 674 and 19032, 741 and 1162.
constexpr int64_t REREADS_MAX = 128 * 128;
template <typename Key>
constexpr int DIGITS = (8 * (int)sizeof(Key) + WIDE_BITS - 1) / WIDE_BITS;

template <typename Key>
struct EvictState { // per pool; behind it, per chunk: {all, any} of Key, counts above and at the prefix
  uint32_t hist[DIGITS<Key>][WIDE_BINS];
  Key prefix[DIGITS<Key> + 1]; // after the range and after each histogram
  int shift[DIGITS<Key> + 1];
  uint32_t need[DIGITS<Key> + 1], count[DIGITS<Key> + 1]; // still needed of those at the prefix; how many there are
  uint32_t tied;    // candidates collected
  Key tied_key[MAX_TIED];
  uint32_t tied_idx[MAX_TIED];
};
template <typename Key>
struct ChunkState {
  Key all, any, tied_all, tied_any;
  uint32_t g, e;
};
template <typename Key>
__host__ __device__ inline int64_t evict_state_bytes(int64_t chunks) {
  return ((int64_t)sizeof(EvictState<Key>) + 255) / 256 * 256 + (chunks * (int64_t)sizeof(ChunkState<Key>) + 255) / 256 * 256;
}
template <typename Key>
struct EvictView {
  EvictState<Key>* st;
  ChunkState<Key>* ch;
};
template <typename Key>
__device__ __forceinline__ EvictView<Key> evict_view(const EvictArgs& a, int64_t b) {
  char* p = static_cast<char*>(a.ws) + b * evict_state_bytes<Key>(a.chunks);
  return EvictView<Key>{reinterpret_cast<EvictState<Key>*>(p), reinterpret_cast<ChunkState<Key>*>(p + (sizeof(EvictState<Key>) + 255) / 256 * 256)};
}

template <typename W>
struct Chunk {
  typedef typename KeyOf<W>::type Key;
  Key key[CHUNK_PER];
  uint32_t free_bits;
  __device__ __forceinline__ void load(const EvictArgs& a, const PoolCut& cut, int64_t b, int64_t j0) {
    const W* w = static_cast<const W*>(a.weights) + b * a.M;
    free_bits = 0;
#pragma unroll
    for (int i = 0; i < CHUNK_PER; ++i) {
      const int64_t j = j0 + i * 1024 + threadIdx.x;
      key[i] = j < cut.L ? order_key(w[j]) : (Key)0;
      free_bits |= (uint32_t)(j >= cut.lo && j < cut.hi) << i;
    }
  }
};

template <typename W>
__global__ __launch_bounds__(1024) void pool_evict_range_kernel(EvictArgs a) {
  typedef typename KeyOf<W>::type Key;
  const int64_t b = blockIdx.y, c = blockIdx.x;
  const PoolCut cut = pool_cut(a, b);
  const EvictView<Key> v = evict_view<Key>(a, b);
  for (int64_t i = c * 1024 + threadIdx.x; i < a.levels * WIDE_BINS; i += a.chunks * 1024) (&v.st->hist[0][0])[i] = 0;
  if (c == 0 && threadIdx.x == 0) v.st->tied = 0;
  Chunk<W> k;
  k.load(a, cut, b, c * CHUNK);
  Key all = ~(Key)0, any = 0;
#pragma unroll
  for (int i = 0; i < CHUNK_PER; ++i)
    if ((k.free_bits >> i) & 1) {
      all &= k.key[i];
      any |= k.key[i];
    }
  __shared__ Key sh[2][16];
  all = block_reduce(all, sh[0], key_and<Key>);
  any = block_reduce(any, sh[1], key_or<Key>);
  if (threadIdx.x == 0) {
    v.ch[c].all = all;
    v.ch[c].any = any;
  }
}

// What is known of a pool's prefix before launch `level` (1, 2 ...: a histogram; behind them: collecting): from the launch
// before, and written for the next by the first chunk.  Nothing is left to decide where need == 0 or every candidate at the prefix stays.
template <typename Key>
struct Prefix {
  Key prefix;
  int shift;
  uint32_t need, count;
};
template <typename Key, bool FIRST>
__device__ __forceinline__ Prefix<Key> advance_prefix(const EvictArgs& a, const EvictView<Key>& v, const PoolCut& cut, int level, Key (*sh_keys)[16]) {
  Prefix<Key> p;
  if (FIRST) {
    Key all = ~(Key)0, any = 0;
    for (int64_t i = threadIdx.x; i < a.chunks; i += 1024) {
      all &= v.ch[i].all;
      any |= v.ch[i].any;
    }
    all = block_reduce(all, sh_keys[0], key_and<Key>);
    any = block_reduce(any, sh_keys[1], key_or<Key>);
    p.shift = cut.need > 0 ? bits_of<Key>(all ^ any) : 0;
    p.prefix = above(all, p.shift);
    p.need = cut.need;
    p.count = (uint32_t)(cut.hi - cut.lo);
  } else {
    p = Prefix<Key>{v.st->prefix[level - 2], v.st->shift[level - 2], v.st->need[level - 2], v.st->count[level - 2]};
    if (p.shift > 0 && p.need > 0 && p.need < p.count) {
      const int lo = p.shift > WIDE_BITS ? p.shift - WIDE_BITS : 0, width = p.shift - lo;
      const Digit d = wide_digit(v.st->hist[level - 2], p.need);
      p.prefix = (p.prefix << width) | (Key)d.bin;
      p.shift = lo;
      p.need -= d.above;
      p.count = d.count;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    v.st->prefix[level - 1] = p.prefix;
    v.st->shift[level - 1] = p.shift;
    v.st->need[level - 1] = p.need;
    v.st->count[level - 1] = p.count;
  }
  return p;
}

template <typename W, bool FIRST>
__global__ __launch_bounds__(1024) void pool_evict_hist_kernel(EvictArgs a, int level) {
  typedef typename KeyOf<W>::type Key;
  __shared__ uint32_t bins[WIDE_BINS];
  __shared__ Key sh_keys[2][16];
  const int64_t b = blockIdx.y, c = blockIdx.x;
  const PoolCut cut = pool_cut(a, b);
  const EvictView<Key> v = evict_view<Key>(a, b);
  if (!FIRST && level > DIGITS<uint32_t>) { // digits that few pools need: not read where nothing was left to decide a launch ago
    const Prefix<Key> q{v.st->prefix[level - 2], v.st->shift[level - 2], v.st->need[level - 2], v.st->count[level - 2]};
    if (q.shift == 0 || q.need == 0 || q.need == q.count) {
      if (c == 0 && threadIdx.x == 0) {
        v.st->prefix[level - 1] = q.prefix;
        v.st->shift[level - 1] = q.shift;
        v.st->need[level - 1] = q.need;
        v.st->count[level - 1] = q.count;
      }
      return;
    }
  }
  Chunk<W> k;
  k.load(a, cut, b, c * CHUNK);
  const Prefix<Key> p = advance_prefix<Key, FIRST>(a, v, cut, level, sh_keys);
  if (p.shift == 0 || p.need == 0 || p.need == p.count) return;
  __syncthreads();
  for (int i = threadIdx.x; i < WIDE_BINS; i += 1024) bins[i] = 0;
  __syncthreads();
  const int lo = p.shift > WIDE_BITS ? p.shift - WIDE_BITS : 0, width = p.shift - lo;
#pragma unroll
  for (int i = 0; i < CHUNK_PER; ++i)
    if (((k.free_bits >> i) & 1) && above(k.key[i], p.shift) == p.prefix) atomicAdd(&bins[(uint32_t)(k.key[i] >> lo) & ((1u << width) - 1u)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < WIDE_BINS; i += 1024)
    if (bins[i]) atomicAdd(&v.st->hist[level - 1][i], bins[i]);
}

template <typename W>
__global__ __launch_bounds__(1024) void pool_evict_collect_kernel(EvictArgs a) {
  typedef typename KeyOf<W>::type Key;
  __shared__ Key sh_keys[2][16];
  __shared__ uint32_t sh_cnt[2][16];
  const int64_t b = blockIdx.y, c = blockIdx.x;
  const PoolCut cut = pool_cut(a, b);
  const EvictView<Key> v = evict_view<Key>(a, b);
  Chunk<W> k;
  k.load(a, cut, b, c * CHUNK);
  const Prefix<Key> p = advance_prefix<Key, false>(a, v, cut, a.levels + 1, sh_keys);
  const bool open = p.shift > 0 && p.need > 0 && p.need < p.count;
  uint32_t g = 0, e = 0;
  Key all = ~(Key)0, any = 0;
#pragma unroll
  for (int i = 0; i < CHUNK_PER; ++i) {
    const int64_t j = c * CHUNK + i * 1024 + threadIdx.x;
    const bool fr = (k.free_bits >> i) & 1;
    const Key hi = above(k.key[i], p.shift);
    g += j < cut.L && (!fr || (p.need > 0 && hi > p.prefix));
    if (fr && p.need > 0 && hi == p.prefix) {
      e += 1;
      all &= k.key[i];
      any |= k.key[i];
    }
  }
  if (open && p.count <= MAX_TIED) { // uniform; in no particular order, which decides nothing
    __shared__ uint32_t found, base;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    uint32_t at = e > 0 ? atomicAdd(&found, e) : 0;
    __syncthreads();
    if (threadIdx.x == 0) base = found > 0 ? atomicAdd(&v.st->tied, found) : 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CHUNK_PER; ++i)
      if (((k.free_bits >> i) & 1) && above(k.key[i], p.shift) == p.prefix) {
        v.st->tied_key[base + at] = k.key[i];
        v.st->tied_idx[base + at++] = (uint32_t)(c * CHUNK + i * 1024 + threadIdx.x);
      }
  }
  g = wave_sum(g);
  e = wave_sum(e);
  if ((threadIdx.x & 63) == 0) {
    sh_cnt[0][threadIdx.x >> 6] = g;
    sh_cnt[1][threadIdx.x >> 6] = e;
  }
  all = block_reduce(all, sh_keys[0], key_and<Key>);
  any = block_reduce(any, sh_keys[1], key_or<Key>);
  if (threadIdx.x == 0) {
    g = e = 0;
    for (int i = 0; i < 16; ++i) {
      g += sh_cnt[0][i];
      e += sh_cnt[1][i];
    }
    v.ch[c].g = g;
    v.ch[c].e = e;
    v.ch[c].tied_all = all;
    v.ch[c].tied_any = any;
  }
}

template <typename W>
__global__ __launch_bounds__(1024) void pool_evict_put_kernel(EvictArgs a) {
  typedef typename KeyOf<W>::type Key;
  __shared__ uint32_t bins[WIDE_BINS];
  __shared__ Key sh_keys[2][16];
  __shared__ uint32_t sh_sum[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t b = blockIdx.y, c = blockIdx.x, j0 = c * CHUNK;
  const PoolCut cut = pool_cut(a, b);
  const EvictView<Key> v = evict_view<Key>(a, b);
  Prefix<Key> p{v.st->prefix[a.levels], v.st->shift[a.levels], v.st->need[a.levels], v.st->count[a.levels]};
  Chunk<W> k;
  k.load(a, cut, b, j0);
  // candidates before this chunk that stay, or are at the prefix; whether all at the prefix are the same
  auto add = [](uint32_t x, uint32_t y) { return x + y; };
  uint32_t g0 = 0, e0 = 0;
  Key all = ~(Key)0, any = 0;
  for (int64_t i = tid; i < a.chunks; i += 1024) {
    if (i < c) {
      g0 += v.ch[i].g;
      e0 += v.ch[i].e;
    }
    all &= v.ch[i].tied_all;
    any |= v.ch[i].tied_any;
  }
  g0 = block_reduce(g0, sh_sum[0], add);
  e0 = block_reduce(e0, sh_sum[1], add);
  all = block_reduce(all, sh_keys[0], key_and<Key>);
  any = block_reduce(any, sh_keys[1], key_or<Key>);
  bool open = p.shift > 0 && p.need > 0 && p.need < p.count;
  bool by_place = false; // ties are cut by their keys and places instead of by their number
  if (open && all == any) {
    p.shift = 0; // the first `need` of equal weights
    p.prefix = all;
    open = false;
  }
  Key tie_prefix = 0;
  uint32_t place_prefix = 0;
  int tie_shift = 0, place_shift = 32;
  if (open && p.count <= MAX_TIED) { // a candidate a thread: the other digits of their keys, then those of their places
    const bool in = tid < (int)p.count;
    const Key kk = in ? v.st->tied_key[tid] : (Key)0;
    const uint32_t place = in ? ~v.st->tied_idx[tid] : 0; // the lower, the better
    uint32_t n = p.need, left = p.count;
    tie_prefix = p.prefix;
    tie_shift = p.shift;
    while (n < left && (tie_shift > 0 || place_shift > 0)) {
      const bool by_key = tie_shift > 0;
      const int from = by_key ? tie_shift : place_shift, lo = from > WIDE_BITS ? from - WIDE_BITS : 0, width = from - lo;
      __syncthreads();
      for (int i = tid; i < WIDE_BINS; i += 1024) bins[i] = 0;
      __syncthreads();
      if (in && above(kk, tie_shift) == tie_prefix && above(place, place_shift) == place_prefix)
        atomicAdd(&bins[(by_key ? (uint32_t)(kk >> lo) : place >> lo) & ((1u << width) - 1u)], 1u);
      __syncthreads();
      const Digit d = wide_digit(bins, n);
      if (by_key) {
        tie_prefix = (tie_prefix << width) | (Key)d.bin;
        tie_shift = lo;
      } else {
        place_prefix = (place_prefix << width) | (uint32_t)d.bin;
        place_shift = lo;
      }
      n -= d.above;
      left = d.count;
    }
    const Key hi = above(kk, tie_shift);
    const bool taken = in && (hi > tie_prefix || (hi == tie_prefix && above(place, place_shift) >= place_prefix));
    const uint32_t taken_before = taken && (int64_t)(uint32_t)~place < j0;
    e0 = block_reduce(taken_before, sh_sum[2], add);
    by_place = true;
  } else if (open) {
    // many candidates that agree in 36 bits and differ below: this workgroup goes through the whole pool, 12 bits at a time,
    // and counts what lies before its chunk.  Slow, and rare: 64-bit weights closer than 2^-26 all over the pool, and one far off
    const Key group = p.prefix;
    const int group_shift = p.shift;
    while (p.shift > 0 && p.need < p.count) {
      const int lo = p.shift > WIDE_BITS ? p.shift - WIDE_BITS : 0, width = p.shift - lo;
      __syncthreads();
      for (int i = tid; i < WIDE_BINS; i += 1024) bins[i] = 0;
      __syncthreads();
      for (int64_t q = 0; q < a.chunks; ++q) {
        Chunk<W> o;
        o.load(a, cut, b, q * CHUNK);
#pragma unroll
        for (int i = 0; i < CHUNK_PER; ++i)
          if (((o.free_bits >> i) & 1) && above(o.key[i], p.shift) == p.prefix) atomicAdd(&bins[(uint32_t)(o.key[i] >> lo) & ((1u << width) - 1u)], 1u);
      }
      __syncthreads();
      const Digit d = wide_digit(bins, p.need);
      p.prefix = (p.prefix << width) | (Key)d.bin;
      p.shift = lo;
      p.need -= d.above;
      p.count = d.count;
    }
    uint32_t more = 0, same = 0; // of the group, before this chunk: above the new prefix, at it
    for (int64_t q = 0; q < c; ++q) {
      Chunk<W> o;
      o.load(a, cut, b, q * CHUNK);
#pragma unroll
      for (int i = 0; i < CHUNK_PER; ++i)
        if (((o.free_bits >> i) & 1) && above(o.key[i], group_shift) == group) {
          more += above(o.key[i], p.shift) > p.prefix;
          same += above(o.key[i], p.shift) == p.prefix;
        }
    }
    g0 += block_reduce(more, sh_sum[2], add);
    e0 = block_reduce(same, sh_sum[3], add);
  }
  uint32_t g_bits = 0, e_bits = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < CHUNK_PER; ++i) {
    const int64_t j = j0 + i * 1024 + tid;
    const bool fr = (k.free_bits >> i) & 1;
    const Key hi = above(k.key[i], p.shift);
    g_bits |= (uint32_t)(j < cut.L && (!fr || (p.need > 0 && hi > p.prefix))) << i;
    bool e = fr && p.need > 0 && hi == p.prefix;
    if (by_place) {
      const Key tie = above(k.key[i], tie_shift);
      e = e && (tie > tie_prefix || (tie == tie_prefix && above(~(uint32_t)j, place_shift) >= place_prefix));
    }
    e_bits |= (uint32_t)e << i;
  }
  put_marked<W, CHUNK_PER>(a, b, j0, g_bits, e_bits, p.need, g0, e0, lane, wave);
  for (int64_t q = cut.keep + c * 1024 + tid; q < a.K; q += a.chunks * 1024) put_nothing<W>(a, b, q);
  if (c == 0 && tid == 0) a.new_lengths[b] = cut.keep;
}

// Payload rows too long for that, of one pool a grid row: 2^log_lanes lanes a row, moved in units; zeros where nothing stayed.
// 64 x 4096 rows of 256 bytes: 20 us (134 MB read and written, 6.6 TB/s); one pool's 4096 rows of 64 bytes: the launch, 4 us.
template <typename Unit>
__global__ __launch_bounds__(256) void pool_gather_kernel(const int64_t* indices, const Unit* src, Unit* dst, int64_t K, int64_t M, int units, int log_lanes) {
  const int64_t b = blockIdx.y;
  const int lanes = 1 << log_lanes, at = threadIdx.x & (lanes - 1), per = 256 >> log_lanes;
  for (int64_t p = (int64_t)blockIdx.x * per + (threadIdx.x >> log_lanes); p < K; p += (int64_t)gridDim.x * per) {
    const int64_t j = indices[b * K + p];
    const Unit* s = src + (b * M + (j < 0 ? 0 : j)) * units;
    Unit* d = dst + (b * K + p) * units;
    for (int u = at; u < units; u += lanes) d[u] = j < 0 ? Unit{} : s[u];
  }
}
template <typename Unit>
void gather_launch(const int64_t* indices, const void* src, void* dst, int64_t pools, int64_t K, int64_t M, int64_t row_bytes, hipStream_t st) {
  const int64_t units = row_bytes / (int64_t)sizeof(Unit);
  int log_lanes = 0;
  while (log_lanes < 8 && ((int64_t)1 << log_lanes) < units) ++log_lanes;
  const int64_t per = 256 >> log_lanes, blocks = (K + per - 1) / per;
  hipLaunchKernelGGL(pool_gather_kernel<Unit>, dim3((unsigned)(blocks < 65536 ? blocks : 65536), (unsigned)pools), dim3(256), 0, st, indices,
                     static_cast<const Unit*>(src), static_cast<Unit*>(dst), K, M, (int)units, log_lanes);
}

// Waves a row in the one-pass kernels, and groups (workgroups); the kernels' comments have both sides of each rule.
struct WeightPlan {
  bool one_pass;
  int waves, groups;
};
WeightPlan weight_plan(int64_t pools, int64_t R, int64_t M, int dtype) {
  auto clamp = [](int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); };
  if (M <= 64 * PER_LANE) {
    return WeightPlan{true, 1, (int)clamp((R + TEAMS - 1) / TEAMS, 1, clamp(512 / (pools > 0 ? pools : 1), 1, 512))};
  }
  if (M <= 64 * team_waves(dtype) * PER_LANE) {
    const int waves = M <= 256 * PER_LANE ? 4 : team_waves(dtype);
    const int64_t want = 4096 / waves; // workgroups that occupy the chip
    return WeightPlan{true, waves, (int)clamp(want / (pools > 0 ? pools : 1), 1, clamp((R + 3) / 4, 1, 1024))};
  }
  return WeightPlan{false, 4, 1};
}
int column_groups(int64_t pools, int64_t R, int64_t M, int dtype) {
  const int64_t tile = 256 * (dtype == GPX_DTYPE_F64 ? 4 : 8), tiles = (M + tile - 1) / tile * (pools > 0 ? pools : 1);
  int64_t g = (1024 + tiles - 1) / tiles; // workgroups that keep the memory busy
  const int64_t most = (R + 15) / 16;
  g = g > most ? most : g;
  return (int)(g < 1 ? 1 : (g > 64 ? 64 : g));
}
int acc_of(int dtype) { return dtype == GPX_DTYPE_F64 ? 8 : 4; }

struct WeightSpace {
  int64_t part, stats, ws, total; // bytes
};
WeightSpace weight_space(int64_t pools, int64_t R, int64_t M, int dtype) {
  const WeightPlan p = weight_plan(pools, R, M, dtype);
  const int groups = p.one_pass ? p.groups : column_groups(pools, R, M, dtype);
  WeightSpace s{};
  s.part = groups > 1 ? round_up64(pools * groups * M * acc_of(dtype), 256) : 0;
  if (!p.one_pass) {
    s.stats = round_up64(2 * pools * R * acc_of(dtype), 256);
    s.ws = row_stats_workspace(pools * R, M, dtype);
  }
  s.total = s.part + s.stats + s.ws;
  return s;
}

template <typename T>
void weights_launch(const WeightArgs& a, const WeightPlan& p, int64_t pools, hipStream_t st) {
  typedef typename Acc<T>::type A;
  if (p.one_pass) {
    const dim3 grid(a.groups, (unsigned)pools);
    const bool dense = a.sc.xc == 1 && (!a.sc.mask || a.sc.mc == 1);
    constexpr int MOST = sizeof(T) == 8 ? 8 : 16;
    if (p.waves == 1)
      hipLaunchKernelGGL(pool_weights_wave_kernel<T>, grid, dim3(TEAMS * 64), 0, st, a);
    else if (p.waves == 4 && dense)
      hipLaunchKernelGGL((pool_weights_kernel<T, 4, true>), grid, dim3(256), 0, st, a);
    else if (p.waves == 4)
      hipLaunchKernelGGL((pool_weights_kernel<T, 4, false>), grid, dim3(256), 0, st, a);
    else if (dense)
      hipLaunchKernelGGL((pool_weights_kernel<T, MOST, true>), grid, dim3(MOST * 64), 0, st, a);
    else
      hipLaunchKernelGGL((pool_weights_kernel<T, MOST, false>), grid, dim3(MOST * 64), 0, st, a);
  } else {
    const int tile = 256 * VecOf<T>::value * col_vecs(sizeof(T));
    const unsigned tiles = (unsigned)((a.sc.M + tile - 1) / tile);
    const dim3 grid(tiles, a.groups, (unsigned)pools);
    if (a.sc.xc == 1 && (!a.sc.mask || a.sc.mc == 1))
      hipLaunchKernelGGL((pool_columns_kernel<T, true>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((pool_columns_kernel<T, false>), grid, dim3(256), 0, st, a);
  }
  if (a.groups > 1) hipLaunchKernelGGL(pool_weights_join_kernel<A>, dim3((a.sc.M + 63) / 64, (unsigned)pools), dim3(256), 0, st, a);
}

// the widest access that a payload's rows allow on both sides
int payload_unit(const void* src, const void* dst, int64_t row_bytes) {
  const uintptr_t al = (uintptr_t)src | (uintptr_t)dst | (uintptr_t)row_bytes;
  return al % 16 == 0 ? 16 : al % 8 == 0 ? 8 : al % 4 == 0 ? 4 : al % 2 == 0 ? 2 : 1;
}
constexpr int64_t HELD_MAX = 16 * 1024; // candidates that one workgroup holds in its registers (both sides: pool_evict_kernel)
int64_t evict_workspace(int dtype, int64_t pools, int64_t M) {
  if (M <= HELD_MAX) return 0;
  const int64_t chunks = (M + CHUNK - 1) / CHUNK;
  return pools * (dtype == GPX_DTYPE_F64 ? evict_state_bytes<uint64_t>(chunks) : evict_state_bytes<uint32_t>(chunks));
}
template <typename W>
void evict_launch(const EvictArgs& a, int64_t pools, hipStream_t st) {
  const dim3 block(1024);
  if (a.M <= HELD_MAX) {
    const dim3 grid((unsigned)pools);
    if (a.M <= 1024)
      hipLaunchKernelGGL((pool_evict_kernel<W, 1>), grid, block, 0, st, a);
    else if (a.M <= 4096)
      hipLaunchKernelGGL((pool_evict_kernel<W, 4>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((pool_evict_kernel<W, 16>), grid, block, 0, st, a);
    return;
  }
  const dim3 grid((unsigned)a.chunks, (unsigned)pools);
  hipLaunchKernelGGL(pool_evict_range_kernel<W>, grid, block, 0, st, a);
  hipLaunchKernelGGL((pool_evict_hist_kernel<W, true>), grid, block, 0, st, a, 1);
  for (int level = 2; level <= a.levels; ++level) hipLaunchKernelGGL((pool_evict_hist_kernel<W, false>), grid, block, 0, st, a, level);
  hipLaunchKernelGGL(pool_evict_collect_kernel<W>, grid, block, 0, st, a);
  hipLaunchKernelGGL(pool_evict_put_kernel<W>, grid, block, 0, st, a);
}

} // namespace

extern "C" {

int64_t gpx_pool_evict_workspace(int64_t pools, int64_t candidates, int dtype) {
  if (pools < 0 || pools > 65535 || candidates < 0 || candidates > POOL_MAX || (dtype != GPX_DTYPE_F64 && dtype != GPX_DTYPE_F32)) return -1;
  return evict_workspace(dtype, pools, candidates);
}

int64_t gpx_pool_weights_workspace(int64_t pools, int64_t rows, int64_t candidates, int dtype) {
  if (!pool_sizes_hold(pools, rows, candidates) || pools > 65535 || dtype < GPX_DTYPE_F64 || dtype > GPX_DTYPE_F16) return -1;
  return weight_space(pools, rows, candidates, dtype).total;
}

int gpx_pool_weights(gpx_ctx* ctx, const gpx_scores* scores, const void* d_row_weights, const void* d_weights, double decay,
                     void* d_out, void* d_workspace, int64_t workspace_bytes, void* stream) {
  if (!ctx || ctx->device < 0) return -1;
  WeightArgs a{};
  GPX_TRY(pool_scores_view(ctx, scores, &a.sc, "gpx_pool_weights"));
  if (scores->pools > 65535) return bad_arg(ctx, "gpx_pool_weights: more than 65535 pools");
  if (!(decay >= 0 && decay < INFINITY)) return bad_arg(ctx, "gpx_pool_weights: the decay must be finite and not negative");
  if (scores->pools == 0 || a.sc.M == 0) return 0;
  if (!d_out) return bad_arg(ctx, "gpx_pool_weights: null output");
  const WeightPlan p = weight_plan(scores->pools, a.sc.R, a.sc.M, scores->dtype);
  const WeightSpace s = weight_space(scores->pools, a.sc.R, a.sc.M, scores->dtype);
  if (s.total > 0 && (!d_workspace || workspace_bytes < s.total))
    return bad_arg(ctx, "gpx_pool_weights: workspace too small (gpx_pool_weights_workspace)");
  a.row_weights = d_row_weights;
  a.weights = decay == 0.0 ? nullptr : d_weights;
  a.out = d_out;
  a.part = d_workspace;
  a.stats = static_cast<char*>(d_workspace) + s.part;
  a.parts = static_cast<char*>(d_workspace) + s.part + s.stats;
  a.splits = 1;
  a.decay = decay;
  a.groups = p.one_pass ? p.groups : column_groups(scores->pools, a.sc.R, a.sc.M, scores->dtype);
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!p.one_pass && a.sc.rows > 0)
    GPX_TRY(launch_row_stats(ctx, a.sc, scores->dtype, a.row_weights, const_cast<void*>(a.stats), const_cast<void*>(a.parts), &a.splits, st));
  switch (scores->dtype) {
    case GPX_DTYPE_F64: weights_launch<double>(a, p, scores->pools, st); break;
    case GPX_DTYPE_F32: weights_launch<float>(a, p, scores->pools, st); break;
    case GPX_DTYPE_BF16: weights_launch<bf16_t>(a, p, scores->pools, st); break;
    default: weights_launch<f16_t>(a, p, scores->pools, st); break;
  }
  GPX_HIP(ctx, hipGetLastError());
  return 0;
}

int gpx_pool_evict(gpx_ctx* ctx, int dtype, int64_t pools, int64_t candidates, const void* d_weights, const void* d_lengths,
                   int lengths_64, int64_t lengths_stride, int64_t budget, int64_t first, int64_t recent, int64_t* d_indices,
                   int64_t* d_new_lengths, void* d_weights_out, int npayload, const void* const* d_payload,
                   void* const* d_payload_out, const int64_t* payload_row_bytes, void* d_workspace, int64_t workspace_bytes,
                   void* stream) {
  if (!ctx || ctx->device < 0) return -1;
  if (dtype != GPX_DTYPE_F64 && dtype != GPX_DTYPE_F32) return bad_arg(ctx, "gpx_pool_evict: weights are float64 or float32");
  if (pools < 0 || candidates < 0 || pools > 65535 || candidates > POOL_MAX)
    return bad_arg(ctx, "gpx_pool_evict: sizes");
  if (budget < 1 || budget > INT32_MAX) return bad_arg(ctx, "gpx_pool_evict: the budget must be positive");
  if (first < 0 || recent < 0 || first > budget || recent > budget - first) return bad_arg(ctx, "gpx_pool_evict: first + recent exceed the budget");
  if (npayload < 0 || npayload > 16) return bad_arg(ctx, "gpx_pool_evict: at most 16 payload arrays");
  if (pools == 0) return 0;
  if ((!d_weights && candidates > 0) || !d_indices || !d_new_lengths || !d_weights_out) return bad_arg(ctx, "gpx_pool_evict: null pointer");
  if (npayload > 0 && (!d_payload || !d_payload_out || !payload_row_bytes)) return bad_arg(ctx, "gpx_pool_evict: null payload arrays");
  for (int i = 0; i < npayload; ++i) {
    if (payload_row_bytes[i] < 0 || payload_row_bytes[i] > INT32_MAX) return bad_arg(ctx, "gpx_pool_evict: payload row size");
    if (payload_row_bytes[i] > 0 && ((!d_payload[i] && candidates > 0) || !d_payload_out[i])) return bad_arg(ctx, "gpx_pool_evict: null payload");
  }
  EvictArgs a{};
  a.weights = d_weights;
  a.lengths = d_lengths;
  a.len64 = lengths_64;
  a.ls = lengths_stride;
  a.M = candidates;
  a.K = budget;
  a.first = first;
  a.recent = recent;
  a.indices = d_indices;
  a.new_lengths = d_new_lengths;
  a.out = d_weights_out;
  a.ws = d_workspace;
  a.chunks = (candidates + CHUNK - 1) / CHUNK;
  a.levels = dtype == GPX_DTYPE_F64 && pools * a.chunks * a.chunks > REREADS_MAX ? DIGITS<uint64_t> : DIGITS<uint32_t>;
  for (int i = 0; i < npayload; ++i) {
    const int64_t rb = payload_row_bytes[i];
    if (rb == 0 || rb > FUSED_ROW_BYTES) continue;
    const int unit = payload_unit(d_payload[i], d_payload_out[i], rb);
    a.pay[a.npay++] = Payload{static_cast<const char*>(d_payload[i]), static_cast<char*>(d_payload_out[i]), (int)rb, unit == 2 ? 1 : unit};
  }
  const int64_t need = evict_workspace(dtype, pools, candidates);
  if (need > 0 && (!d_workspace || workspace_bytes < need)) return bad_arg(ctx, "gpx_pool_evict: workspace too small (gpx_pool_evict_workspace)");
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == GPX_DTYPE_F64)
    evict_launch<double>(a, pools, st);
  else
    evict_launch<float>(a, pools, st);
  for (int i = 0; i < npayload; ++i) {
    const int64_t rb = payload_row_bytes[i];
    if (rb <= FUSED_ROW_BYTES) continue;
    switch (payload_unit(d_payload[i], d_payload_out[i], rb)) {
      case 16: gather_launch<Unit16>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st); break;
      case 8: gather_launch<uint64_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st); break;
      case 4: gather_launch<uint32_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st); break;
      case 2: gather_launch<uint16_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st); break;
      default: gather_launch<uint8_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st); break;
    }
  }
  GPX_HIP(ctx, hipGetLastError());
  return 0;
}

// Device scratch of the context and blocking copies on its stream: what the binding stages host arrays through.
int gpx_scratch(gpx_ctx* ctx, int64_t bytes, void** d_out) {
  if (!ctx || ctx->device < 0) return -1;
  if (bytes < 0 || !d_out) return bad_arg(ctx, "gpx_scratch");
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  GPX_HIP(ctx, hipStreamSynchronize(ctx->stream));
  GPX_HIP(ctx, ctx->pool_scratch.ensure((size_t)(bytes > 0 ? bytes : 1)));
  *d_out = ctx->pool_scratch.p;
  return 0;
}
int gpx_upload(gpx_ctx* ctx, void* d_dst, const void* src, int64_t bytes) {
  if (!ctx || ctx->device < 0) return -1;
  if (bytes < 0 || (bytes > 0 && (!d_dst || !src))) return bad_arg(ctx, "gpx_upload");
  if (bytes == 0) return 0;
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  GPX_HIP(ctx, hipMemcpyAsync(d_dst, src, (size_t)bytes, hipMemcpyHostToDevice, ctx->stream));
  GPX_HIP(ctx, hipStreamSynchronize(ctx->stream));
  return 0;
}
int gpx_download(gpx_ctx* ctx, void* dst, const void* d_src, int64_t bytes) {
  if (!ctx || ctx->device < 0) return -1;
  if (bytes < 0 || (bytes > 0 && (!dst || !d_src))) return bad_arg(ctx, "gpx_download");
  if (bytes == 0) return 0;
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  GPX_HIP(ctx, hipMemcpyAsync(dst, d_src, (size_t)bytes, hipMemcpyDeviceToHost, ctx->stream));
  GPX_HIP(ctx, hipStreamSynchronize(ctx->stream));
  return 0;
}
void* gpx_stream(gpx_ctx* ctx) { return ctx ? static_cast<void*>(ctx->stream) : nullptr; }

} // extern "C"
