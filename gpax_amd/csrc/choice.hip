// choice.hip — the softmax policy over a pool of candidates: log probabilities of given choices, entropy, log of the sum of
// exponentials and the best alternatives of every row in ONE pass over the scores, and the gradient of all of them.
//
// Bound by memory for large pools (a score is read once; 3 - 4 fused operations and one exponential each) and by latency for
// small ones: 2048 x 65536 bfloat16, three inputs in turn, take 53 us (5.1 TB/s) without alternatives, 66 with 20 and 88 with 64 of
// them (one input again and again, partly in cache: 45, 63 and 86).  That is 10.8, 15.4 and 17.9 vector instructions a score, which
// occupy the vector units for 75, 82 and 73 % of the time.  1000 x 1024 float64 take 5.4 and, with 8, 8.8 us; 1 x 201 4.0 and,
// with one, 5.6 us, of which an empty launch is 4.  A row is worked on by 1, 4 or 16 waves of one workgroup, or by several
// workgroups whose partial results a second launch joins: as many waves as it takes to occupy the chip, no more (choice_plan).
//
// Alternatives: every wave keeps the best 64 candidates it has met, one per lane, sorted by (score descending, index
// ascending).  The k-th of them is a threshold that few later candidates pass: a step whose largest score does not is left
// with one comparison.  The few that do are inserted one by one (a ballot gives the position, a shift by one lane makes
// room); many at once are sorted across the lanes and merged.  Lists of waves and workgroups are merged the same way, so
// the order in which they arrive decides nothing: equal scores are told apart by their index.
#include "pool.h"

using namespace gpx;

namespace {

constexpr int TOP_MAX = 64;    // alternatives per row: one per lane of a wave
// More alternatives than this: thresholds from 128 or 256 instead of 64 maxima (1000 x 1024 float64 top 64: 12.6 us against 23.0;
// top 20 9.6 from 64, 10.3 from more; 65536 x 1024 bfloat16 86 and 108).
constexpr int LONG_LIST = 24;
// More newcomers than this in one vector are sorted and merged instead of being inserted one by one (1000 x 1024 float64: top 1
// 7.8 us, always sorted 9.0; top 20 9.6, always inserted 11.6; top 64 12.6 and 18.4).
constexpr int INSERT_MAX = 10;

struct ChoiceArgs {
  PoolScores sc;
  const int64_t* choices; // rows x C, -1 = filler
  int C;
  int top;
  int splits; // workgroups per row
  const void* row_weights; // rows, or nullptr: a row of weight 0 is not read, and has the statistics of an empty one
  void *logprobs, *entropy, *lse, *stats, *top_logprobs;
  int64_t* top_indices;
  void* ws;
};

// The kernel's arguments as if read from memory here: hides from the compiler that they are the ones it has already.
__device__ __forceinline__ const ChoiceArgs& late_args(const ChoiceArgs&) {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const ChoiceArgs*)(const __attribute__((address_space(4))) ChoiceArgs*)p;
}

// A partial result in the workspace: Partial and the list, of one split of one row
inline int64_t partial_bytes(int acc_size, int top) { return 4 * acc_size + round_up64((int64_t)top * (acc_size + 4), 16); }

__device__ __forceinline__ float read_lane(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
__device__ __forceinline__ uint32_t read_lane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ double read_lane(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}

template <typename A>
__device__ __forceinline__ bool before(A k1, uint32_t i1, A k2, uint32_t i2) {
  return k1 > k2 || (k1 == k2 && i1 < i2);
}

// Bitonic networks over the 64 lanes, best first, unrolled: the stage (SIZE, STRIDE) and all behind it.  From (2, 1) on it
// sorts; from (64, 32) on it sorts what is a bitonic sequence already.  Which lanes keep the better one is a constant of the
// stage: as a literal in the scalar unit it costs no register (21 such masks, kept in registers, spilled).
constexpr uint64_t keep_better(int size, int stride) {
  uint64_t m = 0;
  for (int l = 0; l < 64; ++l)
    if (((l & stride) == 0) == ((l & size) == 0)) m |= (uint64_t)1 << l;
  return m;
}
template <int SIZE, int STRIDE, typename A>
__device__ __forceinline__ void bitonic(A& k, uint32_t& i) {
  constexpr uint64_t KEEP = keep_better(SIZE, STRIDE);
  const A ok = xor_lane<STRIDE>(k);
  const uint32_t oi = xor_lane<STRIDE>(i);
  const bool swap = __builtin_amdgcn_inverse_ballot_w64(__ballot(before(k, i, ok, oi)) ^ KEEP);
  k = swap ? ok : k;
  i = swap ? oi : i;
  if constexpr (STRIDE > 1)
    bitonic<SIZE, STRIDE / 2>(k, i);
  else if constexpr (SIZE < 64)
    bitonic<SIZE * 2, SIZE>(k, i);
}

template <int SIZE, int STRIDE, typename A>
__device__ __forceinline__ void bitonic_values(A& v) {
  constexpr uint64_t KEEP = keep_better(SIZE, STRIDE);
  const A o = xor_lane<STRIDE>(v);
  v = __builtin_amdgcn_inverse_ballot_w64(__ballot(v > o) ^ KEEP) ? o : v;
  if constexpr (STRIDE > 1)
    bitonic_values<SIZE, STRIDE / 2>(v);
  else if constexpr (SIZE < 64)
    bitonic_values<SIZE * 2, SIZE>(v);
}
// The k-th largest of the wave's 64 V values (no NaN), or a little less; -inf if fewer than k exist.  64 values are sorted (21
// exchanges).  More are not moved: it is found bit by bit in integers of their order, from the top, with a comparison a value
// and the counting in the scalar unit; a prefix that exactly k reach ends it.  (Of 64 values that takes longer: 65536 x 1024
// bfloat16 top 8 80 instead of 72 us; of 128, 39 us against 57 for 512 x 65536 float32 top 64.)
__device__ __forceinline__ uint32_t order_word(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint32_t order_word(double v) { // (64 bits: of the high word)
  const uint32_t u = (uint32_t)__double2hiint(v);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float least_of_order(uint32_t t, float) {
  return t <= 0x007fffffu ? neg_inf<float>() : __uint_as_float((t >> 31) ? t & 0x7fffffffu : ~t);
}
__device__ __forceinline__ uint32_t low_order(double v) {
  const uint32_t u = (uint32_t)__double2loint(v);
  return __double2hiint(v) < 0 ? ~u : u;
}
// the next number above v (which is not NaN): x > v is x >= that
__device__ __forceinline__ float next_above(float v) {
  const int u = __float_as_int(v);
  return __int_as_float(v == 0.0f ? 1 : u < 0 ? u - 1 : u + 1);
}
__device__ __forceinline__ double next_above(double v) {
  const long long u = __double_as_longlong(v);
  return __longlong_as_double(v == 0.0 ? 1ll : u < 0 ? u - 1 : u + 1);
}
template <typename A, int V>
__device__ __forceinline__ A kth_of(const A (&v)[V], int k) {
  if constexpr (V == 1) {
    A sorted = v[0];
    bitonic_values<2, 1>(sorted);
    return read_lane(sorted, k - 1);
  }
  uint32_t w[V], t = 0;
  int reach = 64 * V; // how many are at least t
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = order_word(v[i]);
#pragma unroll 1
  for (uint32_t bit = 1u << 31; bit != 0 && reach != k; bit >>= 1) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) c += __popcll(__ballot(w[i] >= (t | bit)));
    if (c >= k) {
      t |= bit;
      reach = c;
    }
  }
  if constexpr (sizeof(A) == 4) {
    return least_of_order(t, 0.0f);
  } else {
    if (t <= 0x000fffffu) return neg_inf<A>();
    const uint32_t hi = (t >> 31) ? t & 0x7fffffffu : ~t;
    uint32_t low = 0;
    if (reach > k + 4) { // values that agree in 32 bits: the same for the low word
      uint32_t l[V];
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = low_order(v[i]);
#pragma unroll 1
      for (uint32_t bit = 1u << 31; bit != 0 && reach != k; bit >>= 1) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += __popcll(__ballot(w[i] > t || (w[i] == t && l[i] >= (low | bit))));
        if (c >= k) {
          low |= bit;
          reach = c;
        }
      }
    }
    return __hiloint2double((int)hi, (int)((t >> 31) ? low : ~low));
  }
}

template <typename A>
struct TopList {
  A key;        // lane l: the l-th best; -inf where there is none
  uint32_t idx; // ... and its index; all ones where there is none
  A thr_key;    // the k-th (uniform)
  uint32_t thr_idx;
  int k;

  __device__ __forceinline__ void init(int k_) {
    key = thr_key = neg_inf<A>();
    idx = thr_idx = 0xffffffffu;
    k = k_;
  }
  __device__ __forceinline__ void rethreshold() {
    thr_key = read_lane(key, k - 1);
    thr_idx = read_lane(idx, k - 1);
  }
  // one sorted list into this one: the better of (mine, other reversed) lane by lane holds the best 64 of both as a bitonic
  // sequence, six exchanges sort it
  __device__ __forceinline__ void merge_sorted(A ck, uint32_t ci, int lane) {
    const A rk = __shfl(ck, 63 - lane);
    const uint32_t ri = __shfl(ci, 63 - lane);
    if (before(rk, ri, key, idx)) {
      key = rk;
      idx = ri;
    }
    bitonic<64, 32>(key, idx);
    rethreshold();
  }
  // one candidate a lane (those that do not pass the threshold are dropped)
  __device__ __forceinline__ void consume(A x, uint32_t j, int lane) {
    const bool pass = x > neg_inf<A>() && before(x, j, thr_key, thr_idx); // NaN never passes
    uint64_t in = __ballot(pass);
    if (in == 0) return;
    if (__popcll(in) > INSERT_MAX) {
      A ck = pass ? x : neg_inf<A>();
      uint32_t ci = pass ? j : 0xffffffffu;
      bitonic<2, 1>(ck, ci);
      if (read_lane(idx, 0) == 0xffffffffu) { // the first ones
        key = ck;
        idx = ci;
        rethreshold();
        return;
      }
      merge_sorted(ck, ci, lane);
      return;
    }
    while (in) {
      const int l = __ffsll((unsigned long long)in) - 1;
      in &= in - 1;
      const A nk = read_lane(x, l);
      const uint32_t ni = read_lane(j, l);
      const bool ahead = before(key, idx, nk, ni);
      const int at = __popcll(__ballot(ahead));
      const A pk = __shfl_up(key, 1);
      const uint32_t pi = __shfl_up(idx, 1);
      if (!ahead) {
        key = lane == at ? nk : pk;
        idx = lane == at ? ni : pi;
      }
    }
    rethreshold();
  }
  // a list that is sorted already
  __device__ __forceinline__ void consume_sorted(A ck, uint32_t ci, int lane) {
    if (__ballot(before(ck, ci, thr_key, thr_idx)) == 0) return;
    if (read_lane(idx, 0) == 0xffffffffu) { // the first one
      key = ck;
      idx = ci;
      rethreshold();
      return;
    }
    merge_sorted(ck, ci, lane);
  }
};

// The candidates that may belong into the list.  Of a step only those at or above a bound are looked at one by one: the list's
// threshold, the threshold of all waves of the row, or, where many lanes (and at least k) hold something better, the k-th
// largest of the lanes' maxima (k candidates reach it, so no other can be among the best k).  What passes waits in LDS until 64
// are together; it is offered 64 at a time, the first 64 with their scores, more than that by their
// index, and those scores are read again from the cache.  A threshold that is not up to date only lets more pass.
template <typename A, int E>
struct WaitingRoom {
  A keys[64];
  uint32_t idx[64 * E + 64];
};
template <typename T, int VEC, int U>
struct Waiting {
  typedef typename Acc<T>::type A;
  static constexpr int GROUP = sizeof(A) == 4 ? 4 : U * VEC; // (of 64 bits the groups' maxima would not fit the registers)
  WaitingRoom<A, U * VEC>& room; // this wave's
  A shared;                      // k candidates of the row reach it
  int count;

  __device__ __forceinline__ void flush(TopList<A>& list, const Row<T>& v, int lane) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int i = 0; i < count; i += 64) {
      A k = neg_inf<A>();
      uint32_t j = 0xffffffffu;
      if (i + lane < count) {
        j = room.idx[i + lane];
        if (i == 0)
          k = room.keys[lane];
        else
          k = to_acc(v.x[j * v.xc]);
      }
      list.consume(k, j, lane);
    }
    __builtin_amdgcn_wave_barrier();
    count = 0;
  }
  __device__ __forceinline__ void step(TopList<A>& list, const Row<T>& v, const A* x, A cm, int j0, int lane) {
    // above the list's own threshold strictly: a score equal to its k-th loses to it, whose index is lower (a wave takes its
    // steps in order); at or above the shared one, whose index may be anything
    const A own = list.thr_key;
    A bound = own >= shared ? next_above(own) : shared; // one comparison a score
    const uint64_t better = __ballot(cm >= bound);
    if (better == 0) return;
    const bool many = __popcll(better) >= (list.k > 32 ? list.k : 32);
    if (many) {
      A kth;
      if (list.k <= LONG_LIST) {
        const A top[1] = {cm == cm ? cm : neg_inf<A>()}; // (NaN: nothing else in this lane)
        kth = kth_of(top, list.k);
      } else { // so many of 64 maxima would be too low a bound: four to a lane
        constexpr int Q = U * VEC / 4;
        A top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = neg_inf<A>();
#pragma unroll
          for (int e = q * Q; e < (q + 1) * Q; ++e) top[q] = fmax(top[q], x[e]);
        }
        kth = kth_of(top, list.k);
      }
      bound = kth > bound ? kth : bound;
    }
    // four scores at a time: most steps hold one or two that pass, and the other groups are left with one comparison
#pragma unroll
    for (int g = 0; g < U * VEC; g += GROUP) {
      if (GROUP < U * VEC) {
        A gm = x[g];
#pragma unroll
        for (int e = g + 1; e < g + GROUP; ++e) gm = fmax(gm, x[e]);
        if (__ballot(gm >= bound) == 0) continue;
      }
#pragma unroll
      for (int e = g; e < g + GROUP; ++e) {
        const bool in = x[e] >= bound;
        const uint64_t mask = __ballot(in);
        if (mask) {
          const int at = count + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
          if (in) {
            room.idx[at] = (uint32_t)(j0 + (e / VEC) * 64 * VEC + lane * VEC + e % VEC);
            if (at < 64) room.keys[at] = x[e];
          }
          count += __popcll(mask);
        }
      }
    }
    if (many || count >= 64) flush(list, v, lane); // (many: the threshold will be much better)
  }
};

// What the waves of a workgroup tell each other: maxima, and at the end statistics, and their lists in the front of their waiting
// rooms, which are empty then (LDS decides how many workgroups a CU holds: with 1 KB more for 256 maxima, 7 instead of 8 of
// those with 4 waves, and 2048 x 65536 bfloat16 top 20 takes 81 instead of 74 us).
template <typename A, int W>
struct WaveShare {
  Stats<A> st[W];
  A cells[W > 1 ? 2 : 1][W > 1 ? 128 : 1]; // two in turn: all waves have read one when they meet over the other
};
// A threshold for all waves: the k-th largest of 64 (for long lists 128) maxima, each over all that some lanes of one wave have
// met, so that k candidates of the row reach it.  (Merging the waves' lists for it, one after the other in one wave while the
// others waited, let fewer pass and cost three times as much: 512 x 65536 float32 top 20 took 67 us.)
template <int CELLS, typename A, int W>
__device__ __forceinline__ A common_threshold(A most, int k, WaveShare<A, W>& sh, int turn, int wave, int lane) {
  constexpr int LANES = 64 * W / CELLS; // of a cell
  if constexpr (LANES > 1) most = fmax(most, xor_lane<1>(most));
  if constexpr (LANES > 2) most = fmax(most, xor_lane<2>(most));
  if constexpr (LANES > 4) most = fmax(most, xor_lane<4>(most));
  if constexpr (LANES > 8) most = fmax(most, xor_lane<8>(most));
  static_assert(LANES >= 1 && LANES <= 16, "xor over 16 lanes");
  if (lane % LANES == 0) sh.cells[turn][wave * (64 / LANES) + lane / LANES] = most;
  __syncthreads();
  A top[CELLS / 64];
#pragma unroll
  for (int i = 0; i < CELLS / 64; ++i) top[i] = sh.cells[turn][i * 64 + lane];
  return kth_of(top, k);
}

// (x - m) / T - log s.  Not through powers of two: a lowest score overflows there.  A difference of a whole range overflows too,
// and need not once it is divided.
template <typename A>
__device__ __forceinline__ A log_prob(A x, A m, A T, A log_s) {
  const A d = x - m;
  return (d == neg_inf<A>() ? x / T - m / T : d / T) - log_s;
}

// What a row's statistics are turned into, by a team of `size` threads of which this one is `at`; the list by its wave.
template <typename T>
__device__ __forceinline__ void finish_row(const ChoiceArgs& a, int64_t row, int64_t b, int64_t r, const Stats<typename Acc<T>::type>& st, int at,
                                           int size) {
  typedef typename Acc<T>::type A;
  const A log2s = log2_acc(st.s), log_s = ln2<A>() * log2s, T_row = row_temperature<A>(a.sc, b, r);
  if (at == 0) {
    if (a.entropy) static_cast<A*>(a.entropy)[row] = stats_entropy(st, log2s);
    if (a.lse) static_cast<A*>(a.lse)[row] = st.m / T_row + log_s;
    if (a.stats) {
      static_cast<A*>(a.stats)[2 * row] = st.m;
      static_cast<A*>(a.stats)[2 * row + 1] = log2s;
    }
  }
  if (a.C > 0) {
    const Row<T> v = row_view<T>(a.sc, b, r);
    for (int q = at; q < a.C; q += size) {
      const int64_t j = a.choices[row * a.C + q];
      A lp = (A)0; // a filler
      if (j >= a.sc.M || j < -1) {
        lp = (A)NAN; // no candidate of this pool: never read
      } else if (j >= 0) {
        const A x = row_at(v, (int)j);
        lp = x == neg_inf<A>() ? x : log_prob(x, st.m, T_row, log_s);
      }
      static_cast<A*>(a.logprobs)[row * a.C + q] = lp;
    }
  }
}
template <typename A>
__device__ __forceinline__ void finish_top(const ChoiceArgs& a, int64_t row, int64_t b, int64_t r, const Stats<A>& st, const TopList<A>& list, int lane) {
  if (lane >= a.top) return;
  const bool there = list.idx != 0xffffffffu;
  a.top_indices[row * a.top + lane] = there ? (int64_t)list.idx : -1;
  static_cast<A*>(a.top_logprobs)[row * a.top + lane] =
      there ? log_prob(list.key, st.m, row_temperature<A>(a.sc, b, r), ln2<A>() * log2_acc(st.s)) : neg_inf<A>();
}

// Joins the statistics and lists of the W waves of a workgroup: log2 W rounds, each wave with the one `half` above it.
template <typename A, int W, bool TOP, int E>
__device__ __forceinline__ void join_waves(Stats<A>& st, TopList<A>& list, A c, WaitingRoom<A, E>* rooms, WaveShare<A, W>& sh, int wave, int lane) {
#pragma unroll 1
  for (int half = W / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      if (lane == 0) sh.st[wave] = st;
      if (TOP) {
        rooms[wave].keys[lane] = list.key;
        rooms[wave].idx[lane] = list.idx;
      }
    }
    __syncthreads();
    if (wave < half) {
      st = stats_join(st, sh.st[wave + half], c);
      if (TOP) list.consume_sorted(rooms[wave + half].keys[lane], rooms[wave + half].idx[lane], lane);
    }
  }
}

// Vectors that a lane has in flight: a step of 1024 candidates, or, for pools of at most 256 (512 of 16 bits), one of that
// size: less code to fetch, which is most of what a launch of a few rows spends its time on (1 x 100 float64 top 1: 5.7 us
// instead of 7.3; 20000 x 256 float32 top 1: 16.6 instead of 21.6).
template <typename T>
struct StepOf {
  static constexpr int wide = 16 / VecOf<T>::value, narrow = sizeof(T) == 8 ? 2 : 1;
};

template <typename T, int WAVES, bool TOP, int U>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64, sizeof(T) == 8 || WAVES != 4 ? 1 : 8) void choice_rows_kernel(ChoiceArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value;
  __shared__ WaitingRoom<A, U * VEC> sh_room[TOP ? (WAVES == 1 ? 4 : WAVES) : 1];
  __shared__ WaveShare<A, WAVES> sh_share;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
  if (row >= a.sc.rows) return; // WAVES == 1: whole waves, and no barrier below
  const int64_t b = (uint32_t)row / (uint32_t)a.sc.R, r = row - b * a.sc.R; // at most 2^25 rows
  const A c = temperature_scale(row_temperature<A>(a.sc, b, r));
  Row<T> v = row_view<T>(a.sc, b, r);
  if (!TOP && a.row_weights && static_cast<const A*>(a.row_weights)[row] == (A)0) v.n = 0;
  Stats<A> st = stats_empty<A>();
  TopList<A> list;
  if (TOP) list.init(a.top);
  // candidates are numbered in 32 bits: a pool ends 2^20 short of 2^31, and no stride (2^18 at most) is longer than that
  const int step = 64 * VEC * U;
  const int first = WAVES == 1 ? 0 : ((int)blockIdx.y * WAVES + wave) * step;
  const int stride = WAVES == 1 ? step : a.splits * WAVES * step;
  const int steps = (int)(((uint32_t)v.n + (uint32_t)stride - 1) / (uint32_t)stride); // the same for all waves of the row's workgroup: they meet at barriers
  Waiting<T, VEC, U> waiting{sh_room[TOP ? wave : 0], neg_inf<A>(), 0};
  A most = neg_inf<A>(); // that this lane has met
  int turn = 0;
  for (int i = 0; i < steps; ++i) {
    const int j0 = first + i * stride;
    A x[U * VEC], cm = neg_inf<A>();
    if (j0 < v.n) {
      load_step<T, VEC, U>(v, j0, 64 * VEC, lane * VEC, x);
      cm = x[0];
#pragma unroll
      for (int e = 1; e < U * VEC; ++e) cm = fmax(cm, x[e]);
      stats_add<A, U * VEC>(st, x, cm, c);
    }
    if constexpr (TOP && WAVES > 1) {
      // a threshold of the whole row at steps 1, 2, 4 ...: between two of them about k candidates of the row pass it
      most = fmax(most, cm);
      if (((i + 1) & i) == 0) {
        waiting.shared = list.k <= LONG_LIST ? common_threshold<64>(most, list.k, sh_share, turn, wave, lane)
                                             : common_threshold<128>(most, list.k, sh_share, turn, wave, lane);
        turn ^= 1;
      }
    }
    if constexpr (TOP)
      if (j0 < v.n) waiting.step(list, v, x, cm, j0, lane);
  }
  if constexpr (TOP) waiting.flush(list, v, lane);
  st = stats_wave(st, c);
  const ChoiceArgs& z = late_args(a); // what follows reads its arguments anew: held over the steps they were spilled
  if constexpr (WAVES > 1) {
    __syncthreads();
    join_waves<A, WAVES, TOP>(st, list, c, sh_room, sh_share, wave, lane);
  }
  if (WAVES == 1 || z.splits == 1) {
    if (WAVES == 1) {
      finish_row<T>(z, row, b, r, st, lane, 64);
    } else {
      __shared__ Stats<A> sh;
      if (threadIdx.x == 0) sh = st;
      __syncthreads();
      finish_row<T>(z, row, b, r, sh, threadIdx.x, WAVES * 64);
    }
    if (TOP && (WAVES == 1 || wave == 0)) finish_top(z, row, b, r, st, list, lane);
  } else if (wave == 0) {
    char* at = static_cast<char*>(z.ws) + (row * z.splits + blockIdx.y) * (4 * (int64_t)sizeof(A) + (((int64_t)z.top * (sizeof(A) + 4) + 15) / 16 * 16));
    if (lane == 0) *reinterpret_cast<Partial<A>*>(at) = Partial<A>{st.m, st.s, st.t, (A)0};
    if (TOP && lane < z.top) {
      reinterpret_cast<A*>(at + 4 * sizeof(A))[lane] = list.key;
      reinterpret_cast<uint32_t*>(at + 4 * sizeof(A) + z.top * sizeof(A))[lane] = list.idx;
    }
  }
}

// One workgroup per row: the partial results of its splits, dealt to the waves.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES * 64) void choice_join_kernel(ChoiceArgs a) {
  typedef typename Acc<T>::type A;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const int64_t b = (uint32_t)row / (uint32_t)a.sc.R, r = row - b * a.sc.R; // at most 2^25 rows
  const A c = temperature_scale(row_temperature<A>(a.sc, b, r));
  const int64_t bytes = 4 * (int64_t)sizeof(A) + (((int64_t)a.top * (sizeof(A) + 4) + 15) / 16 * 16);
  const char* base = static_cast<const char*>(a.ws) + row * a.splits * bytes;
  Stats<A> st = stats_empty<A>();
  TopList<A> list;
  if (TOP) list.init(a.top);
  for (int s = wave; s < a.splits; s += WAVES) {
    const Partial<A> p = *reinterpret_cast<const Partial<A>*>(base + s * bytes);
    st = stats_join(st, Stats<A>{p.m, p.s, p.t}, c);
    if (TOP) {
      A k = neg_inf<A>();
      uint32_t i = 0xffffffffu;
      if (lane < a.top) {
        k = reinterpret_cast<const A*>(base + s * bytes + 4 * sizeof(A))[lane];
        i = reinterpret_cast<const uint32_t*>(base + s * bytes + 4 * sizeof(A) + a.top * sizeof(A))[lane];
      }
      list.consume_sorted(k, i, lane);
    }
  }
  __shared__ WaveShare<A, WAVES> sh_share;
  __shared__ WaitingRoom<A, 0> sh_room[TOP ? WAVES : 1];
  join_waves<A, WAVES, TOP>(st, list, c, sh_room, sh_share, wave, lane);
  __shared__ Stats<A> sh;
  if (threadIdx.x == 0) sh = st;
  __syncthreads();
  finish_row<T>(a, row, b, r, sh, threadIdx.x, WAVES * 64);
  if (TOP && wave == 0) finish_top(a, row, b, r, st, list, lane);
}

// Gradient with respect to the scores of  sum g_lp log p(choice) + g_h entropy + g_lse lse + sum g_top log p(alternative):
//   d / d z_j = p_j (g_lse - G - g_h (log p_j + entropy)) + sum over the choices and alternatives that are j of their g,
// G = the sum of all g_lp and g_top that count (a filler, or a choice that may not be made, has no gradient), / T.
// One wave per stretch of one row: elementwise given the row's statistics, so a score is read and a gradient written once.
// The choices that fall into a stretch are found by a ballot and added in their order by the lane that holds the candidate:
// the same choice twice gives the same bits every time.  Bound by memory: 1152 x 16381 float32 30 us, 256 x
// 65536 float64 52 us (5.1 TB/s read and written), 2048 x 32768 bfloat16 59 us (4.5 TB/s).
struct GradArgs {
  PoolScores sc;
  const int64_t* choices;
  int C;
  const void *logprobs, *g_logprobs;
  const int64_t* top_indices;
  int top;
  const void *g_top, *entropy, *stats, *g_entropy, *g_lse;
  void* grad; // rows x M, contiguous
  int stretches;
};

template <typename T>
__global__ __launch_bounds__(256) void choice_grad_kernel(GradArgs a) {
  typedef typename Acc<T>::type A;
  constexpr int VEC = VecOf<T>::value;
  constexpr int U = sizeof(T) == 8 ? 4 : 2;
  constexpr int E = VEC * U;
  const int lane = threadIdx.x & 63;
  const int64_t unit = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = unit / a.stretches;
  if (row >= a.sc.rows) return;
  const int j0 = (int)(unit - row * a.stretches) * (64 * E);
  const int64_t b = (uint32_t)row / (uint32_t)a.sc.R, r = row - b * a.sc.R; // at most 2^25 rows
  const Row<T> v = row_view<T>(a.sc, b, r);
  A x[E];
  load_step<T, VEC, U>(v, j0, 64 * VEC, lane * VEC, x);
  const A Tm = row_temperature<A>(a.sc, b, r);
  const A c = temperature_scale(Tm), inv_T = (A)1 / Tm;
  const A m = static_cast<const A*>(a.stats)[2 * row], log2s = static_cast<const A*>(a.stats)[2 * row + 1];
  const A h = a.g_entropy ? static_cast<const A*>(a.entropy)[row] : (A)0;
  const A gh = a.g_entropy ? static_cast<const A*>(a.g_entropy)[row] : (A)0;
  A add[E];
#pragma unroll
  for (int e = 0; e < E; ++e) add[e] = (A)0;
  A G = (A)0;
  auto gather = [&](const int64_t* idx, const A* g, const A* lp, int n) {
    for (int q0 = 0; q0 < n; q0 += 64) {
      const int q = q0 + lane;
      int64_t j = -1;
      A gq = (A)0;
      if (q < n) {
        j = idx[q];
        gq = g[q];
        if (j < 0 || j >= a.sc.M || (lp && lp[q] == neg_inf<A>())) {
          j = -1;
          gq = (A)0;
        }
      }
      G += gq;
      const bool here = j >= j0 && j < j0 + 64 * E;
      for (uint64_t in = __ballot(here); in; in &= in - 1) {
        const int l = __ffsll((unsigned long long)in) - 1;
        const int off = __builtin_amdgcn_readlane((int)(j - j0), l);
        const A gv = read_lane(gq, l);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (off == (e / VEC) * 64 * VEC + lane * VEC + e % VEC) add[e] += gv;
      }
    }
  };
  if (a.g_logprobs)
    gather(a.choices + row * a.C, static_cast<const A*>(a.g_logprobs) + row * a.C, static_cast<const A*>(a.logprobs) + row * a.C, a.C);
  if (a.g_top) gather(a.top_indices + row * a.top, static_cast<const A*>(a.g_top) + row * a.top, nullptr, a.top);
  G = wave_sum(G);
  const A base = (a.g_lse ? static_cast<const A*>(a.g_lse)[row] : (A)0) - G;
  T* out = static_cast<T*>(a.grad) + row * a.sc.M;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const A xe = x[u * VEC + e];
      const A w = (xe - m) * c - log2s;
      const A g = (exp2_acc(w) * (base - gh * (ln2<A>() * not_below_low(w) + h)) + add[u * VEC + e]) * inv_T;
      from_acc(xe == neg_inf<A>() ? (A)0 : g, o.v[e]);
    }
    const int j = j0 + u * 64 * VEC + lane * VEC;
    if (j + VEC <= a.sc.M) {
      *reinterpret_cast<Pack<T, VEC>*>(out + j) = o;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (j + e < a.sc.M) out[j + e] = o.v[e];
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------

// Waves per row (1, 4 or 16) and workgroups per row.  Enough waves to occupy the chip (TARGET: 16 of the 32 that a CU holds;
// with 32, 1024 x 16384 float32 take 15.7 instead of 13.6 us, with 8, 2048 x 65536 bfloat16 62 instead of 47), but none with less than a step to do: a row shorter than that is one wave's, however few rows there are (1000 x 1024 float64
// 5 us as one wave a row).  One workgroup a row up to 16 waves spares the second launch (4 us) and most of the lists' joining;
// beyond that up to 64 workgroups share one, more than 32 only if their waves have two steps each (8 x 262144 float64 top 64:
// 32 take 15.2 us and 8.7 to join, 64 take 13.7 and 11.9; 2 x 1048576 float32: 26.4 and 7.0 against 18.1 and 9.5).
struct ChoicePlan {
  int waves, splits;
};
ChoicePlan choice_plan(int64_t rows, int64_t M) {
  constexpr int64_t TARGET = 4096;
  const int64_t steps = (M + 1023) / 1024;
  int64_t want = rows > 0 ? (TARGET + rows - 1) / rows : 1;
  if (want > steps) want = steps;
  if (want <= 1) return ChoicePlan{1, 1};
  if (want <= 4) return ChoicePlan{4, 1};
  if (want <= 16) return ChoicePlan{16, 1};
  int64_t splits = (want + 3) / 4;
  const int64_t most = steps < 32 * 8 ? 32 : (steps > 64 * 8 ? 64 : steps / 8);
  if (splits > most) splits = most;
  return ChoicePlan{4, (int)splits};
}

template <typename T, bool TOP>
void choice_launch(const ChoiceArgs& a, ChoicePlan p, hipStream_t st, bool join) {
  const unsigned rows = (unsigned)a.sc.rows;
  constexpr int U = StepOf<T>::wide, UN = StepOf<T>::narrow;
  if (p.waves == 1) {
    if (a.sc.M <= 64 * VecOf<T>::value * UN)
      hipLaunchKernelGGL((choice_rows_kernel<T, 1, TOP, UN>), dim3((rows + 3) / 4), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((choice_rows_kernel<T, 1, TOP, U>), dim3((rows + 3) / 4), dim3(256), 0, st, a);
  } else if (p.waves == 16) {
    hipLaunchKernelGGL((choice_rows_kernel<T, 16, TOP, U>), dim3(rows), dim3(1024), 0, st, a);
  } else {
    hipLaunchKernelGGL((choice_rows_kernel<T, 4, TOP, U>), dim3(rows, p.splits), dim3(256), 0, st, a);
    if (p.splits > 1 && join) hipLaunchKernelGGL((choice_join_kernel<T, 16, TOP>), dim3(rows), dim3(1024), 0, st, a);
  }
}
template <typename T>
void choice_launch(const ChoiceArgs& a, ChoicePlan p, hipStream_t st, bool join) {
  if (a.top > 0)
    choice_launch<T, true>(a, p, st, join);
  else
    choice_launch<T, false>(a, p, st, join);
}
void choice_launch(int dtype, const ChoiceArgs& a, ChoicePlan p, hipStream_t st, bool join = true) {
  switch (dtype) {
    case GPX_DTYPE_F64: return choice_launch<double>(a, p, st, join);
    case GPX_DTYPE_F32: return choice_launch<float>(a, p, st, join);
    case GPX_DTYPE_BF16: return choice_launch<bf16_t>(a, p, st, join);
    default: return choice_launch<f16_t>(a, p, st, join);
  }
}
int acc_size(int dtype) { return dtype == GPX_DTYPE_F64 ? 8 : 4; }
int64_t choice_workspace(int64_t rows, int64_t M, int dtype, int top) {
  const ChoicePlan p = choice_plan(rows, M);
  return p.splits == 1 ? 0 : rows * p.splits * partial_bytes(acc_size(dtype), top);
}

} // namespace

namespace gpx {

int pool_scores_view(gpx_ctx* ctx, const gpx_scores* x, PoolScores* out, const char* what) {
  auto no = [&](const char* why) { return bad_arg(ctx, (std::string(what) + ": " + why).c_str()); };
  if (!x) return no("null scores");
  if (x->dtype < GPX_DTYPE_F64 || x->dtype > GPX_DTYPE_F16) return no("dtype");
  if (x->pools < 0 || x->rows < 0 || x->candidates < 0) return no("negative size");
  if (x->candidates > POOL_MAX) return no("more than 2^31 - 2^20 candidates");
  if (!pool_sizes_hold(x->pools, x->rows, x->candidates)) return no("more than 2^25 rows");
  if (x->pools * x->rows > 0 && x->candidates > 0 && !x->d_scores) return no("null scores");
  if (!x->d_temperatures && !(x->temperature > 0 && x->temperature < INFINITY)) return no("the temperature must be positive and finite");
  out->x = x->d_scores;
  out->mask = x->d_mask;
  out->lengths = x->d_lengths;
  out->temps = x->d_temperatures;
  out->xb = x->scores_stride[0];
  out->xr = x->scores_stride[1];
  out->xc = x->scores_stride[2];
  out->mb = x->mask_stride[0];
  out->mr = x->mask_stride[1];
  out->mc = x->mask_stride[2];
  out->lb = x->lengths_stride[0];
  out->lr = x->lengths_stride[1];
  out->tb = x->temperatures_stride[0];
  out->tr = x->temperatures_stride[1];
  out->R = x->rows;
  out->rows = x->pools * x->rows;
  out->M = (int)x->candidates;
  out->len64 = x->lengths_64;
  out->temperature = x->temperature;
  return 0;
}

int64_t row_stats_workspace(int64_t rows, int64_t M, int dtype) { return choice_workspace(rows, M, dtype, 0); }
int launch_row_stats(gpx_ctx* ctx, const PoolScores& sc, int dtype, const void* d_row_weights, void* d_stats, void* d_parts, int* splits,
                     hipStream_t st) {
  ChoiceArgs a{};
  const ChoicePlan p = choice_plan(sc.rows, sc.M);
  a.sc = sc;
  a.splits = p.splits;
  a.row_weights = d_row_weights;
  a.stats = d_stats;
  a.ws = d_parts;
  *splits = p.splits;
  choice_launch(dtype, a, p, st, false);
  GPX_HIP(ctx, hipGetLastError());
  return 0;
}

} // namespace gpx

extern "C" {

int64_t gpx_choice_workspace(int64_t pools, int64_t rows, int64_t candidates, int dtype, int top) {
  if (!pool_sizes_hold(pools, rows, candidates) || top < 0 || top > TOP_MAX || dtype < GPX_DTYPE_F64 || dtype > GPX_DTYPE_F16) return -1;
  return choice_workspace(pools * rows, candidates, dtype, top);
}

int gpx_choice_logprobs(gpx_ctx* ctx, const gpx_scores* scores, const int64_t* d_choices, int64_t nchoices, int top,
                        void* d_logprobs, void* d_entropy, void* d_logsumexp, void* d_stats, int64_t* d_top_indices,
                        void* d_top_logprobs, void* d_workspace, int64_t workspace_bytes, void* stream) {
  if (!ctx || ctx->device < 0) return -1;
  ChoiceArgs a{};
  GPX_TRY(pool_scores_view(ctx, scores, &a.sc, "gpx_choice_logprobs"));
  if (nchoices < 0 || nchoices > INT32_MAX - 1024) return bad_arg(ctx, "gpx_choice_logprobs: number of choices");
  if (top < 0 || top > TOP_MAX) return bad_arg(ctx, "gpx_choice_logprobs: top must be 0..64");
  if (a.sc.rows == 0) return 0;
  if (nchoices > 0 && (!d_choices || !d_logprobs)) return bad_arg(ctx, "gpx_choice_logprobs: null choices");
  if (top > 0 && (!d_top_indices || !d_top_logprobs)) return bad_arg(ctx, "gpx_choice_logprobs: null alternatives");
  if (!d_entropy || !d_logsumexp || !d_stats) return bad_arg(ctx, "gpx_choice_logprobs: null output");
  const ChoicePlan p = choice_plan(a.sc.rows, a.sc.M);
  const int64_t need = choice_workspace(a.sc.rows, a.sc.M, scores->dtype, top);
  if (need > 0 && (!d_workspace || workspace_bytes < need)) return bad_arg(ctx, "gpx_choice_logprobs: workspace too small (gpx_choice_workspace)");
  a.choices = d_choices;
  a.C = (int)nchoices;
  a.top = top;
  a.splits = p.splits;
  a.logprobs = d_logprobs;
  a.entropy = d_entropy;
  a.lse = d_logsumexp;
  a.stats = d_stats;
  a.top_indices = d_top_indices;
  a.top_logprobs = d_top_logprobs;
  a.ws = d_workspace;
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  choice_launch(scores->dtype, a, p, static_cast<hipStream_t>(stream));
  GPX_HIP(ctx, hipGetLastError());
  return 0;
}

int gpx_choice_logprobs_grad(gpx_ctx* ctx, const gpx_scores* scores, const int64_t* d_choices, int64_t nchoices,
                             const void* d_logprobs, const void* d_grad_logprobs, int top, const int64_t* d_top_indices,
                             const void* d_grad_top, const void* d_entropy, const void* d_stats, const void* d_grad_entropy,
                             const void* d_grad_logsumexp, void* d_grad_scores, void* stream) {
  if (!ctx || ctx->device < 0) return -1;
  GradArgs a{};
  GPX_TRY(pool_scores_view(ctx, scores, &a.sc, "gpx_choice_logprobs_grad"));
  if (nchoices < 0 || nchoices > INT32_MAX - 1024) return bad_arg(ctx, "gpx_choice_logprobs_grad: number of choices");
  if (top < 0 || top > TOP_MAX) return bad_arg(ctx, "gpx_choice_logprobs_grad: top must be 0..64");
  if (a.sc.rows == 0 || a.sc.M == 0) return 0;
  if (!d_stats || !d_grad_scores) return bad_arg(ctx, "gpx_choice_logprobs_grad: null statistics or gradient");
  if (d_grad_logprobs && nchoices > 0 && (!d_choices || !d_logprobs)) return bad_arg(ctx, "gpx_choice_logprobs_grad: null choices");
  if (d_grad_top && top > 0 && !d_top_indices) return bad_arg(ctx, "gpx_choice_logprobs_grad: null alternatives");
  if (d_grad_entropy && !d_entropy) return bad_arg(ctx, "gpx_choice_logprobs_grad: null entropy");
  a.choices = d_choices;
  a.C = (int)nchoices;
  a.logprobs = d_logprobs;
  a.g_logprobs = nchoices > 0 ? d_grad_logprobs : nullptr;
  a.top_indices = d_top_indices;
  a.top = top;
  a.g_top = top > 0 ? d_grad_top : nullptr;
  a.entropy = d_entropy;
  a.stats = d_stats;
  a.g_entropy = d_grad_entropy;
  a.g_lse = d_grad_logsumexp;
  a.grad = d_grad_scores;
  const int per = 64 * (scores->dtype == GPX_DTYPE_F64 || scores->dtype == GPX_DTYPE_F32 ? 8 : 16);
  a.stretches = (a.sc.M + per - 1) / per;
  const int64_t units = a.sc.rows * a.stretches;
  const int64_t groups = (units + 3) / 4, gx = groups < (1 << 22) ? groups : (1 << 22), gy = (groups + gx - 1) / gx;
  if (gy > 65535) return bad_arg(ctx, "gpx_choice_logprobs_grad: too many scores");
  DeviceGuard g(ctx->device);
  GPX_HIP(ctx, g.err);
  const dim3 grid((unsigned)gx, (unsigned)gy), block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (scores->dtype) {
    case GPX_DTYPE_F64: hipLaunchKernelGGL(choice_grad_kernel<double>, grid, block, 0, st, a); break;
    case GPX_DTYPE_F32: hipLaunchKernelGGL(choice_grad_kernel<float>, grid, block, 0, st, a); break;
    case GPX_DTYPE_BF16: hipLaunchKernelGGL(choice_grad_kernel<bf16_t>, grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL(choice_grad_kernel<f16_t>, grid, block, 0, st, a); break;
  }
  GPX_HIP(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
