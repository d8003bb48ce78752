// pool.h — what the operators over a pool of candidates share (choice.hip: the softmax policy and its gradient; pool.hip:
// gathered weights and eviction): the view of a row of scores, the exponential, the running softmax statistics.
//
// A row holds one score per candidate; z_j = x_j / T, p_j = exp(z_j) / sum exp(z_i).  With m = max x and c = log2(e) / T every
// quantity below is held relative to m, in powers of two, so that one multiplication stands between a score and its exponent:
//   s = sum 2^((x_j - m) c),  t = sum 2^((x_j - m) c) (x_j - m) c,  log p_j = ln 2 ((x_j - m) c - log2 s),
//   entropy = ln 2 (log2 s - t / s),  log sum exp z = m / T + ln s.
// x - m is formed before the product: it is exact or nearly so where p is not negligible, whatever the size of the scores.
// Candidates behind the row's length, masked out or of score -inf do not exist for any of this; they are read as -inf by
// SELECTION, so that NaN or infinities in those places never enter the arithmetic.
#pragma once
#include "common.h"

namespace gpx {

struct PoolScores {
  const void* x;
  const uint8_t* mask;  // nullptr: none; nonzero = may be chosen
  const void* lengths;  // nullptr: the whole pool
  const void* temps;    // nullptr: `temperature` for every row; else of the accumulator's type
  int64_t xb, xr, xc;   // strides in elements: pool, row, candidate
  int64_t mb, mr, mc, lb, lr, tb, tr;
  int64_t R;            // rows per pool
  int64_t rows;         // pools * R
  int M;                // candidates
  int len64;            // lengths are int64 (else int32)
  double temperature;
};

struct bf16_t {
  uint16_t v;
};
struct f16_t {
  _Float16 v;
};
// sums and statistics: 64 bits for 64-bit scores, 32 bits for the rest (16-bit scores are exact in 32)
template <typename T>
struct Acc {
  typedef float type;
};
template <>
struct Acc<double> {
  typedef double type;
};
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ float to_acc(bf16_t v) { return __uint_as_float((uint32_t)v.v << 16); }
__device__ __forceinline__ float to_acc(f16_t v) { return (float)v.v; }
// the one rounding of a result to its storage type: to nearest, ties to even
__device__ __forceinline__ void from_acc(double a, double& o) { o = a; }
__device__ __forceinline__ void from_acc(float a, float& o) { o = a; }
__device__ __forceinline__ void from_acc(float a, f16_t& o) { o.v = (_Float16)a; }
__device__ __forceinline__ void from_acc(float a, bf16_t& o) {
  const uint32_t u = __float_as_uint(a);
  o.v = (a != a) ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}

template <typename A>
__device__ __forceinline__ A neg_inf();
template <>
__device__ __forceinline__ float neg_inf<float>() {
  return -INFINITY;
}
// Its high word is hidden from the compiler: as a known constant that lives in a scalar register pair, hipcc (ROCm 7.2) loads
// it with one s_mov_b64, whose literal has 32 bits only, and the value becomes 0 (tests/test_pool.py looks for that).
template <>
__device__ __forceinline__ double neg_inf<double>() {
  int hi = (int)0xfff00000;
  asm("" : "+s"(hi));
  return __hiloint2double(hi, 0);
}

__device__ __forceinline__ float exp2_acc(float w) { return __builtin_amdgcn_exp2f(w); }
// 2^w in 64 bits for w <= 0: n = the nearest integer, r = w - n in [-1/2, 1/2], 2^r by the Taylor series of exp(r ln 2) to
// degree 13 ((ln 2 / 2)^14 / 14! < 5e-18), 2^n by ldexp.  NaN passes; below 2^-1100 the result is 0 (as from -inf).
__device__ __forceinline__ double exp2_acc(double w) {
  w = (w < -1100.0) ? -1100.0 : w;
  const double n = __builtin_rint(w);
  const double y = (w - n) * 0.69314718055994530942;
  double p = 1.0 / 6227020800.0;
  p = fma(p, y, 1.0 / 479001600.0);
  p = fma(p, y, 1.0 / 39916800.0);
  p = fma(p, y, 1.0 / 3628800.0);
  p = fma(p, y, 1.0 / 362880.0);
  p = fma(p, y, 1.0 / 40320.0);
  p = fma(p, y, 1.0 / 5040.0);
  p = fma(p, y, 1.0 / 720.0);
  p = fma(p, y, 1.0 / 120.0);
  p = fma(p, y, 1.0 / 24.0);
  p = fma(p, y, 1.0 / 6.0);
  p = fma(p, y, 0.5);
  p = fma(p, y, 1.0);
  p = fma(p, y, 1.0);
  return __builtin_ldexp(p, (int)n);
}
__device__ __forceinline__ float log2_acc(float v) { return log2f(v); }
__device__ __forceinline__ double log2_acc(double v) { return log2(v); }
template <typename A>
__device__ __forceinline__ A ln2() {
  return (A)0.69314718055994530942;
}

// The value of lane ^ S, without the detour through LDS that a shuffle takes: DPP within rows of 16 lanes, row swaps beyond
// (an exchange of 64-bit keys costs 60 cycles instead of 200; sorting 64 lanes has 21 of them in a row).
template <int S>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
  if constexpr (S == 1) {
    return __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false); // quad_perm 1 0 3 2
  } else if constexpr (S == 2) {
    return __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false); // quad_perm 2 3 0 1
  } else if constexpr (S == 4) { // lanes 0-3 and 8-11 of a row from 4 above, the others from 4 below
    const uint32_t up = __builtin_amdgcn_update_dpp(v, v, 0x104, 0xF, 0x5, false);
    return __builtin_amdgcn_update_dpp(up, v, 0x114, 0xF, 0xA, false);
  } else if constexpr (S == 8) {
    return __builtin_amdgcn_update_dpp(v, v, 0x128, 0xF, 0xF, false); // rotation of 16 by 8
  } else if constexpr (S == 16) { // first: odd rows replaced by the even ones below them; second: the other way round
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __builtin_amdgcn_inverse_ballot_w64(0xFFFF0000FFFF0000ull) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_inverse_ballot_w64(0xFFFFFFFF00000000ull) ? r[0] : r[1];
  }
}
template <int S>
__device__ __forceinline__ float xor_lane(float v) {
  return __uint_as_float(xor_lane<S>(__float_as_uint(v)));
}
template <int S>
__device__ __forceinline__ double xor_lane(double v) {
  return __hiloint2double((int)xor_lane<S>((uint32_t)__double2hiint(v)), (int)xor_lane<S>((uint32_t)__double2loint(v)));
}
template <int S>
__device__ __forceinline__ uint64_t xor_lane(uint64_t v) {
  return ((uint64_t)xor_lane<S>((uint32_t)(v >> 32)) << 32) | xor_lane<S>((uint32_t)v);
}
template <typename V, typename F>
__device__ __forceinline__ V wave_reduce(V v, F f) {
  v = f(v, xor_lane<32>(v));
  v = f(v, xor_lane<16>(v));
  v = f(v, xor_lane<8>(v));
  v = f(v, xor_lane<4>(v));
  v = f(v, xor_lane<2>(v));
  return f(v, xor_lane<1>(v));
}
template <typename V>
__device__ __forceinline__ V wave_max(V v) {
  return wave_reduce(v, [](V x, V y) { return fmax(x, y); });
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
  return wave_reduce(v, [](V x, V y) { return x + y; });
}

template <typename A>
__device__ __forceinline__ A row_temperature(const PoolScores& sc, int64_t b, int64_t r) {
  return sc.temps ? static_cast<const A*>(sc.temps)[b * sc.tb + r * sc.tr] : (A)sc.temperature;
}
// log2(e) / T.  T must be positive and finite: anything else makes the row NaN.
template <typename A>
__device__ __forceinline__ A temperature_scale(A T) {
  const A c = (A)1.4426950408889634074 / T;
  return (T > (A)0 && T < (A)INFINITY && c < (A)INFINITY) ? c : (A)NAN;
}
__device__ __forceinline__ int row_length(const PoolScores& sc, int64_t b, int64_t r) {
  if (!sc.lengths) return sc.M;
  const int64_t at = b * sc.lb + r * sc.lr;
  const int64_t n = sc.len64 ? static_cast<const int64_t*>(sc.lengths)[at] : (int64_t)static_cast<const int32_t*>(sc.lengths)[at];
  return n < 0 ? 0 : (n > sc.M ? sc.M : (int)n);
}

template <typename T>
struct Row {
  const T* x;
  const uint8_t* mask;
  int64_t xc, mc;
  int n;
};
template <typename T>
__device__ __forceinline__ Row<T> row_view(const PoolScores& sc, int64_t b, int64_t r) {
  Row<T> v;
  v.x = static_cast<const T*>(sc.x) + b * sc.xb + r * sc.xr;
  v.mask = sc.mask ? sc.mask + b * sc.mb + r * sc.mr : nullptr;
  v.xc = sc.xc;
  v.mc = sc.mc;
  v.n = row_length(sc, b, r);
  return v;
}
template <typename T>
__device__ __forceinline__ typename Acc<T>::type row_at(const Row<T>& v, int j) {
  typedef typename Acc<T>::type A;
  if (j < 0 || j >= v.n) return neg_inf<A>();
  if (v.mask && !v.mask[j * v.mc]) return neg_inf<A>();
  return to_acc(v.x[j * v.xc]);
}

// VEC scores in one load.  The type asks for the alignment of a single score only: rows of odd length and views that start
// anywhere take the same path (the hardware loads four words from any word address; a misaligned one costs a second line).
template <typename T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[VEC];
};
template <int VEC>
struct __attribute__((packed, aligned(1))) MaskPack {
  uint8_t v[VEC];
};
template <typename T>
struct VecOf {
  static constexpr int value = 16 / (int)sizeof(T);
};

// U vectors of VEC scores per lane: x[u * VEC + e] is candidate j0 + u * span + lane_j + e; -inf where there is none.
// `span` (the team's lanes * VEC) and j0 are uniform over the team.  Addresses are clamped into the row instead of being
// guarded one by one, so that every load of a step is in flight at once; they are a uniform base and a small offset per lane.
template <typename T, int VEC, int U>
__device__ __forceinline__ void load_step(const Row<T>& v, int j0, int span, int lane_j, typename Acc<T>::type* x) {
  typedef typename Acc<T>::type A;
  const bool dense = v.xc == 1 && (!v.mask || v.mc == 1);
  if (dense && j0 + U * span <= v.n) {
    Pack<T, VEC> p[U];
    const T* at = v.x + j0;
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = *reinterpret_cast<const Pack<T, VEC>*>(at + (uint32_t)(u * span + lane_j));
    if (v.mask) {
      MaskPack<VEC> q[U];
      const uint8_t* mat = v.mask + j0;
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = *reinterpret_cast<const MaskPack<VEC>*>(mat + (uint32_t)(u * span + lane_j));
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u * VEC + e] = q[u].v[e] ? to_acc(p[u].v[e]) : neg_inf<A>();
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u * VEC + e] = to_acc(p[u].v[e]);
    }
    return;
  }
  if (dense && v.n >= VEC) {
    // the end of the row: vectors that would cross it read the row's last VEC scores instead (and are dropped) ...
    const int last = v.n - VEC, base = j0 < last ? j0 : last;
    Pack<T, VEC> p[U];
    MaskPack<VEC> q[U];
    const T* at = v.x + base;
    const uint8_t* mat = v.mask + base;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * span + lane_j;
      const uint32_t off = (uint32_t)((j < last ? j : last) - base);
      p[u] = *reinterpret_cast<const Pack<T, VEC>*>(at + off);
      if (v.mask) q[u] = *reinterpret_cast<const MaskPack<VEC>*>(mat + off);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = j0 + u * span + lane_j <= last;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[u * VEC + e] = in && (!v.mask || q[u].v[e]) ? to_acc(p[u].v[e]) : neg_inf<A>();
    }
    // ... and the one vector of one lane that the end falls into is read score by score
    if (v.n > j0 && (v.n - j0) % VEC != 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int first = j0 + u * span;
        if (v.n < first || v.n >= first + span) continue; // uniform
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int j = first + lane_j + e, off = j < v.n ? j : v.n - 1;
          const A a = to_acc(v.x[off]);
          const bool there = !v.mask || v.mask[off] != 0;
          if (first + lane_j > last && j < v.n) x[u * VEC + e] = there ? a : neg_inf<A>();
        }
      }
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int j = j0 + u * span + lane_j + e;
      A a = neg_inf<A>();
      if (v.n > 0) { // uniform
        const int64_t at = j < v.n ? j : v.n - 1;
        a = to_acc(v.x[at * v.xc]);
        if (j >= v.n || (v.mask && !v.mask[at * v.mc])) a = neg_inf<A>();
      }
      x[u * VEC + e] = a;
    }
}

// The same in two halves, for a kernel that has the next row on its way while it works on one: `load` starts the loads,
// `decode` makes the scores of them.  DENSE: candidates (and mask bytes) side by side.  Pools of VEC candidates or more.
template <typename T, int VEC, int U, bool DENSE>
struct RawStep {
  typedef typename Acc<T>::type A;
  Pack<T, VEC> p[U];
  MaskPack<VEC> q[U];

  // vectors that would cross the end of the POOL (of M candidates) read its last ones instead
  __device__ __forceinline__ void load(const Row<T>& v, int M, int span, int lane_j) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * span >= v.n) continue; // uniform: nothing of it exists
      const int j = u * span + lane_j, off = j < M - VEC ? j : M - VEC;
      if (DENSE) {
        p[u] = *reinterpret_cast<const Pack<T, VEC>*>(v.x + (uint32_t)off);
        if (v.mask) q[u] = *reinterpret_cast<const MaskPack<VEC>*>(v.mask + (uint32_t)off);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          p[u].v[e] = v.x[(off + e) * v.xc];
          if (v.mask) q[u].v[e] = v.mask[(off + e) * v.mc];
        }
      }
    }
  }
  // x[u * VEC + e] is candidate min(u * span + lane_j, M - VEC) + e
  __device__ __forceinline__ void decode(bool masked, int n, int M, int span, int lane_j, A* x) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if ((u + 1) * span <= n && !masked) { // uniform: all of it is there
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u * VEC + e] = to_acc(p[u].v[e]);
        continue;
      }
      const int j = u * span + lane_j, off = j < M - VEC ? j : M - VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // a candidate belongs to the lane whose own vector it lies in
        const bool in = u * span < n && off + e >= j && off + e < n && (!masked || q[u].v[e]);
        x[u * VEC + e] = in ? to_acc(p[u].v[e]) : neg_inf<A>();
      }
    }
  }
};

// ---- running statistics of a row --------------------------------------------------------------------------------------
template <typename A>
struct Stats {
  A m, s, t;
};
template <typename A>
__device__ __forceinline__ Stats<A> stats_empty() {
  return Stats<A>{neg_inf<A>(), (A)0, (A)0};
}
template <typename A>
__device__ __forceinline__ A finite_max(A m) { // the reference point of a row that has nothing yet: anything finite
  return m == neg_inf<A>() ? (A)0 : m;
}
// 2^low = 0.  Exponents that are multiplied by a power are kept above it, so that 0 * -inf does not arise: from candidates
// that do not exist, and from scores so low (a type's lowest value) that the exponent overflows.
template <typename A>
__device__ __forceinline__ A not_below_low(A w) {
  const A low = sizeof(A) == 8 ? (A)-1e6 : (A)-1e4;
  return w > low ? w : low;
}
// a's sums, taken relative to `to` (>= a.m) instead of a.m
template <typename A>
__device__ __forceinline__ void stats_rebase(Stats<A>& a, A to, A c) {
  const A d = not_below_low((a.m - to) * c);
  const A f = exp2_acc(d);
  a.t = (a.m == neg_inf<A>()) ? a.t : f * (a.t + a.s * d); // nothing gathered yet: both sums are 0 (or NaN, and stay it)
  a.s = (a.m == neg_inf<A>()) ? a.s : f * a.s;
  a.m = to;
}
template <typename A, int E>
__device__ __forceinline__ void stats_add(Stats<A>& a, const A* x, A cm, A c) {
  const A to = a.m > cm ? a.m : cm;
  if (to != a.m) stats_rebase(a, to, c);
  const A ref = finite_max(to);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const A w = (x[e] - ref) * c;
    const A p = exp2_acc(w);
    a.s += p;
    a.t = fma(p, not_below_low(w), a.t);
  }
}
template <typename A>
__device__ __forceinline__ Stats<A> stats_join(Stats<A> a, Stats<A> b, A c) {
  const A to = a.m > b.m ? a.m : b.m;
  if (a.m != to) stats_rebase(a, to, c);
  if (b.m != to) stats_rebase(b, to, c);
  return Stats<A>{to, a.s + b.s, a.t + b.t};
}
template <typename A>
__device__ __forceinline__ Stats<A> stats_wave(Stats<A> a, A c) {
  const A to = wave_max(a.m);
  if (a.m != to) stats_rebase(a, to, c);
  a.s = wave_sum(a.s);
  a.t = wave_sum(a.t);
  return a;
}
// what later passes need of a row's statistics: log2 s and the entropy.  A row without candidates: -inf and 0.
template <typename A>
__device__ __forceinline__ A stats_entropy(const Stats<A>& a, A log2s) {
  return a.s == (A)0 ? (A)0 : ln2<A>() * (log2s - a.t / a.s);
}

// A partial result of one split of a row, as choice.hip leaves it (behind it, where there is one, the list of alternatives)
template <typename A>
struct Partial {
  A m, s, t, pad;
};
// m and log2 s of a row from either form; 16 neighbouring lanes work on one row, `at` of them
template <typename A>
__device__ __forceinline__ void row_reference(const void* stats, const void* parts, int splits, int64_t row, A c, int at, A& m, A& log2s) {
  if (splits == 1) { // uniform
    m = static_cast<const A*>(stats)[2 * row];
    log2s = static_cast<const A*>(stats)[2 * row + 1];
    return;
  }
  const Partial<A>* p = static_cast<const Partial<A>*>(parts) + row * splits;
  Stats<A> st = stats_empty<A>();
  for (int i = at; i < splits; i += 16) st = stats_join(st, Stats<A>{p[i].m, p[i].s, (A)0}, c);
  st = stats_join(st, Stats<A>{xor_lane<8>(st.m), xor_lane<8>(st.s), (A)0}, c);
  st = stats_join(st, Stats<A>{xor_lane<4>(st.m), xor_lane<4>(st.s), (A)0}, c);
  st = stats_join(st, Stats<A>{xor_lane<2>(st.m), xor_lane<2>(st.s), (A)0}, c);
  st = stats_join(st, Stats<A>{xor_lane<1>(st.m), xor_lane<1>(st.s), (A)0}, c);
  m = st.m;
  log2s = log2_acc(st.s);
}

// pool.hip / choice.hip, host side
constexpr int64_t POOL_MAX = INT32_MAX - (1 << 20), ROWS_MAX = 1 << 25; // candidates of a pool; rows of all pools
inline bool pool_sizes_hold(int64_t pools, int64_t rows, int64_t candidates) {
  return pools >= 0 && rows >= 0 && candidates >= 0 && candidates <= POOL_MAX && (rows == 0 || pools <= ROWS_MAX / rows);
}
int pool_scores_view(gpx_ctx* ctx, const gpx_scores* x, PoolScores* out, const char* what);
struct DeviceGuard { // the caller's current device comes back whatever happens
  int before = -1;
  bool switched = false;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) {
      err = hipSetDevice(device);
      switched = err == hipSuccess;
    }
  }
  ~DeviceGuard() {
    if (switched) (void)hipSetDevice(before);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};
// Statistics of every row, pass one of pool_weights over pools too long for a workgroup (choice.hip): rows x {m, log2 s} in
// d_stats if *splits comes back as 1, else partial results of *splits parts of each row in d_parts; rows of weight 0 as empty ones
int launch_row_stats(gpx_ctx* ctx, const PoolScores& sc, int dtype, const void* d_row_weights, void* d_stats, void* d_parts, int* splits,
                     hipStream_t st);
int64_t row_stats_workspace(int64_t rows, int64_t M, int dtype);

} // namespace gpx
