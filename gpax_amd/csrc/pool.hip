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
  const void* stats;       // rows x {m, log2 s} (column pass)
  double decay;
  int groups;
};

constexpr int PER_LANE = 16; // candidates a lane owns in the one-pass kernel
constexpr int TEAMS = 8;     // rows at a time of a workgroup whose teams are single waves
// the largest team: 16 sums and 16 scores of 64 bits do not fit the 128 registers that 16 waves leave each lane
inline int team_waves(int dtype) { return dtype == GPX_DTYPE_F64 ? 8 : 16; }

// a finished sum of candidates j .. j + VEC: straight to the output, or to this group's partial sums
template <typename A, int VEC>
__device__ __forceinline__ void store_sums(const WeightArgs& a, int64_t b, int group, int64_t j, const A* acc) {
  const int64_t M = a.sc.M;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (j + e >= M) return;
    if (a.groups > 1) {
      static_cast<A*>(a.part)[(b * a.groups + group) * M + j + e] = acc[e];
    } else {
      const A old = a.weights ? (A)a.decay * static_cast<const A*>(a.weights)[b * M + j + e] : (A)0;
      static_cast<A*>(a.out)[b * M + j + e] = old + acc[e];
    }
  }
}

// One pass: a team of WAVES waves per row, NTEAMS teams per workgroup.
template <typename T, int WAVES, int NTEAMS>
__global__ __launch_bounds__(WAVES* NTEAMS * 64) void pool_weights_kernel(WeightArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value, U = PER_LANE / VEC, LANES = WAVES * 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wave / WAVES, at = threadIdx.x - team * LANES;
  const int64_t b = blockIdx.y;
  __shared__ A red[2][2][WAVES];
  A acc[PER_LANE];
#pragma unroll
  for (int e = 0; e < PER_LANE; ++e) acc[e] = (A)0;
  int flip = 0;
  for (int64_t r = (int64_t)blockIdx.x * NTEAMS + team; r < a.sc.R; r += (int64_t)a.groups * NTEAMS) {
    const A u = a.row_weights ? static_cast<const A*>(a.row_weights)[b * a.sc.R + r] : (A)1;
    if (u == (A)0) continue; // uniform over the team
    const A c = temperature_scale(row_temperature<A>(a.sc, b, r));
    const Row<T> v = row_view<T>(a.sc, b, r);
    A x[PER_LANE];
    load_step<T, VEC, U>(v, 0, LANES * VEC, at * VEC, x);
    A m = x[0];
#pragma unroll
    for (int e = 1; e < PER_LANE; ++e) m = fmax(m, x[e]);
    m = wave_max(m);
    if (WAVES > 1) { // two buffers: a row's values are overwritten two barriers after they were read
      if ((threadIdx.x & 63) == 0) red[flip][0][wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmax(m, red[flip][0][w]);
    }
    const A ref = finite_max(m);
    A s = (A)0;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) {
      x[e] = exp2_acc((x[e] - ref) * c);
      s += x[e];
    }
    s = wave_sum(s);
    if (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) red[flip][1][wave] = s;
      __syncthreads();
      s = (A)0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += red[flip][1][w];
      flip ^= 1;
    }
    if (s == (A)0) continue; // nothing in this row may be chosen
    const A f = u / s;
    if (f != f) { // NaN for what may be chosen, nothing for what may not
      load_step<T, VEC, U>(v, 0, LANES * VEC, at * VEC, x);
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) acc[e] += x[e] == neg_inf<A>() ? (A)0 : f;
    } else {
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) acc[e] = fma(x[e], f, acc[e]);
    }
  }
  if (NTEAMS > 1) { // the teams' sums in the order of the teams, into the first one's registers
    __shared__ A sum[LANES * PER_LANE];
    for (int t = NTEAMS - 1; t > 0; --t) {
      if (team == t) {
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) sum[e * LANES + at] = (t == NTEAMS - 1 ? (A)0 : sum[e * LANES + at]) + acc[e];
      }
      __syncthreads();
    }
    if (team != 0) return;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) acc[e] += sum[e * LANES + at];
  }
#pragma unroll
  for (int w = 0; w < U; ++w) store_sums<A, VEC>(a, b, blockIdx.x, (int64_t)w * LANES * VEC + at * VEC, acc + w * VEC);
}

// Second pass over longer pools: the rows' statistics are known, a workgroup sums 256 x VEC candidates over its share of rows.
template <typename T>
__global__ __launch_bounds__(256) void pool_columns_kernel(WeightArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value, ROWS = 4;
  const int64_t b = blockIdx.z;
  const int64_t j0 = (int64_t)blockIdx.x * 256 * VEC;
  const int64_t per = (a.sc.R + a.groups - 1) / a.groups;
  const int64_t r1 = per * (blockIdx.y + 1) < a.sc.R ? per * (blockIdx.y + 1) : a.sc.R;
  A acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = (A)0;
  for (int64_t r = per * blockIdx.y; r < r1; r += ROWS) {
    A x[ROWS][VEC];
    Row<T> v[ROWS];
    bool whole = true; // all of the rows' tile exists: their loads are in flight together
#pragma unroll
    for (int q = 0; q < ROWS; ++q) { // past the last row: that row again, with weight 0
      v[q] = row_view<T>(a.sc, b, r + q < r1 ? r + q : r1 - 1);
      whole = whole && v[q].xc == 1 && (!v[q].mask || v[q].mc == 1) && j0 + 256 * VEC <= v[q].n;
    }
    if (whole) {
      Pack<T, VEC> p[ROWS];
      MaskPack<VEC> k[ROWS];
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        p[q] = *reinterpret_cast<const Pack<T, VEC>*>(v[q].x + j0 + threadIdx.x * VEC);
        if (v[q].mask) k[q] = *reinterpret_cast<const MaskPack<VEC>*>(v[q].mask + j0 + threadIdx.x * VEC);
      }
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[q][e] = !v[q].mask || k[q].v[e] ? to_acc(p[q].v[e]) : neg_inf<A>();
    } else {
#pragma unroll
      for (int q = 0; q < ROWS; ++q) load_step<T, VEC, 1>(v[q], j0, 256 * VEC, threadIdx.x * VEC, x[q]);
    }
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const int64_t rq = r + q < r1 ? r + q : r1 - 1;
      const int64_t row = b * a.sc.R + rq;
      const A u = r + q >= r1 ? (A)0 : a.row_weights ? static_cast<const A*>(a.row_weights)[row] : (A)1;
      if (u == (A)0) continue;
      const A c = temperature_scale(row_temperature<A>(a.sc, b, rq));
      const A m = static_cast<const A*>(a.stats)[2 * row], log2s = static_cast<const A*>(a.stats)[2 * row + 1];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const A p = u * exp2_acc((x[q][e] - m) * c - log2s);
        acc[e] += x[q][e] == neg_inf<A>() ? (A)0 : p;
      }
    }
  }
  store_sums<A, VEC>(a, b, blockIdx.y, j0 + threadIdx.x * VEC, acc);
}

// decay w + the groups' partial sums in their order: 64 candidates per workgroup, the groups dealt to its four waves
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

constexpr int EVICT_PER = 16, EVICT_CHUNK = 1024 * EVICT_PER;

struct EvictArgs {
  const void* weights; // pools x M
  const void* lengths;
  int len64;
  int64_t ls; // stride of lengths
  int64_t M, K, first, recent;
  int64_t* indices; // pools x K
  int64_t* new_lengths;
  void* out; // pools x K
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

struct Digit { // where the need-th largest lies in a histogram, counted from the top
  int bin;
  uint32_t above, count;
};
// 256 bins by one wave: lane l holds bins 4 l .. 4 l + 3
__device__ __forceinline__ Digit find_digit(const uint32_t* hist, uint32_t need, int lane) {
  uint32_t c[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * lane + i];
  uint32_t upto = sum; // of this lane and all above it
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t v = __shfl_down(upto, o);
    if (lane + o < 64) upto += v;
  }
  uint32_t above = upto - sum;
  Digit d{0, 0, 0};
  bool mine = false;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    if (!mine && above < need && need <= above + c[i]) {
      d = Digit{4 * lane + i, above, c[i]};
      mine = true;
    }
    above += c[i];
  }
  const int l = __ffsll((unsigned long long)__ballot(mine)) - 1; // need is at least 1 and at most the total: one lane has it
  d.bin = __builtin_amdgcn_readlane(d.bin, l);
  d.above = (uint32_t)__builtin_amdgcn_readlane((int)d.above, l);
  d.count = (uint32_t)__builtin_amdgcn_readlane((int)d.count, l);
  return d;
}

// One workgroup per pool.  The need-th largest weight is found digit by digit (8 bits, a histogram in LDS each), starting at
// the highest bit in which the weights differ at all and ending as soon as a digit holds exactly what is still needed; a
// second sweep writes what stays, in order.  HELD: the pool fits the workgroup's registers (16384 candidates).
template <typename W, bool HELD>
__global__ __launch_bounds__(1024) void pool_evict_kernel(EvictArgs a) {
  typedef typename KeyOf<W>::type Key;
  constexpr int BITS = sizeof(Key) * 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t b = blockIdx.x;
  const W* w = static_cast<const W*>(a.weights) + b * a.M;
  int64_t L = a.M;
  if (a.lengths) {
    L = a.len64 ? static_cast<const int64_t*>(a.lengths)[b * a.ls] : (int64_t)static_cast<const int32_t*>(a.lengths)[b * a.ls];
    L = L < 0 ? 0 : (L > a.M ? a.M : L);
  }
  const int64_t keep = L < a.K ? L : a.K;
  const int64_t lo_free = L <= a.K ? 0 : a.first, hi_free = L <= a.K ? 0 : L - a.recent; // outside: stays whatever its weight
  uint32_t need = L <= a.K ? 0u : (uint32_t)(a.K - a.first - a.recent);
  const int64_t chunks = HELD ? 1 : (L + EVICT_CHUNK - 1) / EVICT_CHUNK;

  __shared__ uint32_t hist[2][256];
  __shared__ Key sh_and[16], sh_or[16];
  __shared__ uint32_t cnt_g[EVICT_PER * 16], cnt_e[EVICT_PER * 16];
  __shared__ uint32_t run_g, run_e;

  Key key[EVICT_PER];
  auto load = [&](int64_t chunk) {
#pragma unroll
    for (int i = 0; i < EVICT_PER; ++i) {
      const int64_t j = chunk * EVICT_CHUNK + i * 1024 + tid;
      key[i] = j < L ? order_key(w[j]) : (Key)0;
    }
  };
  auto is_free = [&](int64_t chunk, int i) {
    const int64_t j = chunk * EVICT_CHUNK + i * 1024 + tid;
    return j >= lo_free && j < hi_free;
  };
  Key prefix = 0;
  int shift = BITS; // key >> shift against prefix; at BITS nothing is compared
  if (HELD) load(0);
  if (need > 0) {
    Key all = ~(Key)0, any = 0;
    for (int64_t ch = 0; ch < chunks; ++ch) {
      if (!HELD) load(ch);
#pragma unroll
      for (int i = 0; i < EVICT_PER; ++i)
        if (is_free(ch, i)) {
          all &= key[i];
          any |= key[i];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      all &= __shfl_xor(all, o);
      any |= __shfl_xor(any, o);
    }
    if (lane == 0) {
      sh_and[wave] = all;
      sh_or[wave] = any;
    }
    if (tid < 256) hist[0][tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      all &= sh_and[i];
      any |= sh_or[i];
    }
    const Key diff = all ^ any;
    shift = diff == 0 ? 0 : BITS - (sizeof(Key) == 8 ? __clzll((long long)diff) : __clz((int)diff));
    prefix = shift < BITS ? all >> shift : (Key)0; // shift == 0: every weight is the same
    int flip = 0;
    while (shift > 0) {
      const int lo = shift > 8 ? shift - 8 : 0, width = shift - lo;
      for (int64_t ch = 0; ch < chunks; ++ch) {
        if (!HELD) load(ch);
#pragma unroll
        for (int i = 0; i < EVICT_PER; ++i)
          if (is_free(ch, i) && (shift >= BITS || (key[i] >> (shift & (BITS - 1))) == prefix))
            atomicAdd(&hist[flip][(uint32_t)(key[i] >> lo) & ((1u << width) - 1u)], 1u);
      }
      __syncthreads();
      const Digit d = find_digit(hist[flip], need, lane);
      flip ^= 1;
      if (tid < 256) hist[flip][tid] = 0;
      prefix = (shift >= BITS ? (Key)0 : prefix << width) | (Key)d.bin;
      need -= d.above;
      shift = lo;
      __syncthreads();
      if (need == d.count) break; // the whole digit stays
    }
  }
  // above the prefix: stays; equal to it: the first `need` in order
  const int64_t base = b * a.K;
  if (tid == 0) run_g = run_e = 0;
  __syncthreads();
  for (int64_t ch = 0; ch < chunks; ++ch) {
    if (!HELD) load(ch);
    uint32_t g_bits = 0, e_bits = 0;
#pragma unroll
    for (int i = 0; i < EVICT_PER; ++i) {
      const int64_t j = ch * EVICT_CHUNK + i * 1024 + tid;
      const bool fr = is_free(ch, i);
      const Key hi = shift >= BITS ? (Key)0 : key[i] >> (shift & (BITS - 1));
      const bool g = j < L && (!fr || hi > prefix), e = fr && need > 0 && hi == prefix;
      const uint64_t bg = __ballot(g), be = __ballot(e);
      if (lane == 0) {
        cnt_g[i * 16 + wave] = (uint32_t)__popcll(bg);
        cnt_e[i * 16 + wave] = (uint32_t)__popcll(be);
      }
      g_bits |= (uint32_t)g << i;
      e_bits |= (uint32_t)e << i;
    }
    __syncthreads();
    if (wave == 0) { // exclusive sums of the 256 counts, in the order of the candidates
      uint32_t g4[4], e4[4], sg = 0, se = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g4[i] = sg;
        e4[i] = se;
        sg += cnt_g[4 * lane + i];
        se += cnt_e[4 * lane + i];
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
      const uint32_t og = run_g, oe = run_e;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cnt_g[4 * lane + i] = og + pg - sg + g4[i];
        cnt_e[4 * lane + i] = oe + pe - se + e4[i];
      }
      if (lane == 63) {
        run_g = og + pg;
        run_e = oe + pe;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EVICT_PER; ++i) {
      const bool g = (g_bits >> i) & 1, e = (e_bits >> i) & 1;
      const uint64_t bg = __ballot(g), be = __ballot(e);
      const uint64_t below = (1ull << lane) - 1;
      const uint32_t ng = cnt_g[i * 16 + wave] + (uint32_t)__popcll(bg & below);
      const uint32_t ne = cnt_e[i * 16 + wave] + (uint32_t)__popcll(be & below);
      if (g || (e && ne < need)) {
        const int64_t j = ch * EVICT_CHUNK + i * 1024 + tid;
        const int64_t pos = base + ng + (ne < need ? ne : need);
        a.indices[pos] = j;
        static_cast<W*>(a.out)[pos] = w[j];
      }
    }
    __syncthreads();
  }
  for (int64_t p = keep + tid; p < a.K; p += 1024) {
    a.indices[base + p] = -1;
    static_cast<W*>(a.out)[base + p] = (W)0;
  }
  if (tid == 0) a.new_lengths[b] = keep;
}

// Payload rows of what stayed: `row` bytes each, moved in units of UNIT bytes; zeros where nothing stayed.
template <typename Unit>
__global__ __launch_bounds__(256) void pool_gather_kernel(const int64_t* indices, const Unit* src, Unit* dst, int64_t total, int64_t K, int64_t M, int units) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / units, u = i - row * units, b = row / K;
    const int64_t j = indices[row];
    Unit v{};
    if (j >= 0) v = src[(b * M + j) * units + u];
    dst[i] = v;
  }
}
struct alignas(16) Unit16 {
  uint32_t v[4];
};
template <typename Unit>
void gather_launch(const int64_t* indices, const void* src, void* dst, int64_t pools, int64_t K, int64_t M, int64_t row_bytes, hipStream_t st) {
  const int64_t units = row_bytes / (int64_t)sizeof(Unit), total = pools * K * units;
  const int64_t blocks = (total + 255) / 256;
  hipLaunchKernelGGL(pool_gather_kernel<Unit>, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st, indices,
                     static_cast<const Unit*>(src), static_cast<Unit*>(dst), total, K, M, (int)units);
}

// Teams that work off a pool's rows in the one-pass kernel, and groups (workgroups) of them.
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
int column_groups(int64_t pools, int64_t R, int64_t M, int vec) {
  const int64_t tiles = (M + 256 * vec - 1) / (256 * vec) * (pools > 0 ? pools : 1);
  int64_t g = (512 + tiles - 1) / tiles; // workgroups that keep the memory busy
  const int64_t most = (R + 15) / 16;
  g = g > most ? most : g;
  return (int)(g < 1 ? 1 : (g > 64 ? 64 : g));
}
int vec_of(int dtype) { return dtype == GPX_DTYPE_F64 ? 2 : dtype == GPX_DTYPE_F32 ? 4 : 8; }
int acc_of(int dtype) { return dtype == GPX_DTYPE_F64 ? 8 : 4; }

struct WeightSpace {
  int64_t part, stats, ws, total; // bytes
};
WeightSpace weight_space(int64_t pools, int64_t R, int64_t M, int dtype) {
  const WeightPlan p = weight_plan(pools, R, M, dtype);
  const int groups = p.one_pass ? p.groups : column_groups(pools, R, M, vec_of(dtype));
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
    if (p.waves == 1)
      hipLaunchKernelGGL((pool_weights_kernel<T, 1, TEAMS>), grid, dim3(TEAMS * 64), 0, st, a);
    else if (p.waves == 4)
      hipLaunchKernelGGL((pool_weights_kernel<T, 4, 1>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((pool_weights_kernel<T, sizeof(T) == 8 ? 8 : 16, 1>), grid, dim3(p.waves * 64), 0, st, a);
  } else {
    const unsigned tiles = (unsigned)((a.sc.M + 256 * VecOf<T>::value - 1) / (256 * VecOf<T>::value));
    hipLaunchKernelGGL(pool_columns_kernel<T>, dim3(tiles, a.groups, (unsigned)pools), dim3(256), 0, st, a);
  }
  if (a.groups > 1) hipLaunchKernelGGL(pool_weights_join_kernel<A>, dim3((a.sc.M + 63) / 64, (unsigned)pools), dim3(256), 0, st, a);
}

} // namespace

extern "C" {

int64_t gpx_pool_weights_workspace(int64_t pools, int64_t rows, int64_t candidates, int dtype) {
  if (pools < 0 || rows < 0 || candidates < 0 || dtype < GPX_DTYPE_F64 || dtype > GPX_DTYPE_F16) return -1;
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
  a.weights = d_weights;
  a.out = d_out;
  a.part = d_workspace;
  a.stats = static_cast<char*>(d_workspace) + s.part;
  a.decay = decay;
  a.groups = p.one_pass ? p.groups : column_groups(scores->pools, a.sc.R, a.sc.M, vec_of(scores->dtype));
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!p.one_pass && a.sc.rows > 0)
    GPX_TRY(launch_row_stats(ctx, a.sc, scores->dtype, const_cast<void*>(a.stats), static_cast<char*>(d_workspace) + s.part + s.stats, st));
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
                   void* const* d_payload_out, const int64_t* payload_row_bytes, void* stream) {
  if (!ctx || ctx->device < 0) return -1;
  if (dtype != GPX_DTYPE_F64 && dtype != GPX_DTYPE_F32) return bad_arg(ctx, "gpx_pool_evict: weights are float64 or float32");
  if (pools < 0 || candidates < 0 || pools > INT32_MAX / 1024 / 4 || candidates > INT32_MAX - 65536)
    return bad_arg(ctx, "gpx_pool_evict: sizes");
  if (budget < 1 || budget > INT32_MAX) return bad_arg(ctx, "gpx_pool_evict: the budget must be positive");
  if (first < 0 || recent < 0 || first + recent > budget) return bad_arg(ctx, "gpx_pool_evict: first + recent exceed the budget");
  if (npayload < 0 || npayload > 16) return bad_arg(ctx, "gpx_pool_evict: at most 16 payload arrays");
  if (pools == 0) return 0;
  if ((!d_weights && candidates > 0) || !d_indices || !d_new_lengths || !d_weights_out) return bad_arg(ctx, "gpx_pool_evict: null pointer");
  for (int i = 0; i < npayload; ++i) {
    if (payload_row_bytes[i] < 0 || payload_row_bytes[i] > INT32_MAX) return bad_arg(ctx, "gpx_pool_evict: payload row size");
    if (payload_row_bytes[i] > 0 && ((!d_payload[i] && candidates > 0) || !d_payload_out[i])) return bad_arg(ctx, "gpx_pool_evict: null payload");
  }
  EvictArgs a{d_weights, d_lengths, lengths_64, lengths_stride, candidates, budget, first, recent, d_indices, d_new_lengths, d_weights_out};
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)pools), block(1024);
  const bool held = candidates <= EVICT_CHUNK;
  if (dtype == GPX_DTYPE_F64) {
    if (held)
      hipLaunchKernelGGL((pool_evict_kernel<double, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((pool_evict_kernel<double, false>), grid, block, 0, st, a);
  } else {
    if (held)
      hipLaunchKernelGGL((pool_evict_kernel<float, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((pool_evict_kernel<float, false>), grid, block, 0, st, a);
  }
  for (int i = 0; i < npayload; ++i) {
    const int64_t rb = payload_row_bytes[i];
    if (rb == 0) continue;
    const uintptr_t al = (uintptr_t)d_payload[i] | (uintptr_t)d_payload_out[i] | (uintptr_t)rb;
    if (al % 16 == 0)
      gather_launch<Unit16>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st);
    else if (al % 8 == 0)
      gather_launch<uint64_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st);
    else if (al % 4 == 0)
      gather_launch<uint32_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st);
    else if (al % 2 == 0)
      gather_launch<uint16_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st);
    else
      gather_launch<uint8_t>(d_indices, d_payload[i], d_payload_out[i], pools, budget, candidates, rb, st);
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
