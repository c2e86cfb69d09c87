// Log probabilities of given tokens, the entropy of the distribution and the
// best alternatives, from rows of logits.
//
// With x a row, M its largest value at index i*, d_i = x_i - M,
//   S = sum_{i != i*} e^{d_i},  T = sum_i e^{d_i} d_i
//   log p_t = d_t - log1p(S),  H = log1p(S) - T / (1 + S)
// S leaves the largest value's own 1 out, so that a confident token's log
// probability keeps its digits (1 + 1e-9 has none in 32 bits).  Values of -inf
// (tokens that are ruled out) have probability 0 and add nothing to H.  (M, S,
// T) of two parts of a row join as
//   M = M1 >= M2, D = M2 - M1, f = e^D:
//   S = S1 + f (S2 + 1),  T = T1 + f (T2 + D (S2 + 1)).
//
// Bound by one read of the logits.  Each wave works on its own: 1024 values of
// one row at a time, 16 in each lane, the next 1024 in flight.  In a lane a
// tournament of 15 comparisons finds the largest value; its 15 losers each cost
// one exponential, so that the largest is left out of S without a test per
// value.  A wave keeps the alternatives it has seen in its first lanes, in
// order; only values that can still be among the row's best, by what the
// work-group's waves have told each other, are looked at one by one.  Rows are
// cut so that a launch has about kGroups work-groups; the last piece of a row to
// end joins them all.
// 1,000 rows of 151,936 bf16 logits (304 MB): 64-69 us, 4.6 TB/s, VALU issue about
// as long; with each wave's list on its own 73, with a search of the work-group
// for each alternative and a barrier a tile 199.  8 f32 rows: 11.0-13.1 us alone
// (the chain load -> statistics -> ticket -> join), among others 4.3-4.7 in some
// processes and 8.4-8.9 in others.
//
// Alternatives are ordered by value, equal ones by index (lower first, -0 and 0
// are equal), NaN below -inf.
#include <algorithm>

#include "fmd_common.h"
#include "fmd_kernels.h"

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64, kPer = 16, kTile = 64 * kPer;
constexpr int kGroups = 512;
constexpr int kMaxTop = 32;
constexpr int kRanked = 1024;   // keys that a join ranks in LDS
// Up to this largest value the rounding of m log2e is at most 2^-12, and 2^-err
// is 1 - err ln2 within (2^-12 ln2)^2 / 2 < 2^-25.
constexpr float kNear = 4096.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Largest and smallest of two, NaN if either is.
__device__ __forceinline__ float top2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float low2(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// m in the logits' units, s and t over exponents in log2 units (t's as well).
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  if (a.m < b.m) {
    const Stat c = a;
    a = b;
    b = c;
  }
  if (b.m == -INFINITY) {   // nothing there, or NaN alone (in s)
    a.s += b.s;
    return a;
  }
  // not below -1000 (2^-1000 is 0, and so is 0 * -1000): the type's lowest value,
  // as a mask, is further from a logit than the product can say
  const float d = top2((b.m - a.m) * kLog2e, -1000.f), f = __builtin_amdgcn_exp2f(d), n = b.s + 1.f;
  a.s += f * n;
  a.t += f * (b.t + d * n);
  return a;
}

// Order of the alternatives as an integer; 0 is below every value's.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t idx) {
  v += 0.f;   // -0 -> 0
  uint32_t b = __builtin_bit_cast(uint32_t, v);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (v != v) b = 0;
  return ((uint64_t)b << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) {
  uint32_t b = (uint32_t)(k >> 32);
  if (b == 0) return NAN;
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __builtin_bit_cast(float, b);
}

// What a piece of a row leaves for the row's join.
struct Part {
  uint64_t keys[kMaxTop];
  uint64_t ms, t;   // Stat's m and s, t
};
__device__ __forceinline__ void put(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Shared {
  uint64_t joined[kMaxTop];
  uint32_t told[kWaves];
  uint64_t wave[2][kWaves];
  Stat stat[kWaves];
  uint32_t ticket;
  uint64_t all[kRanked];            // lists to be joined
};

// Largest of the wave's words, in every lane: DPP steps inside rows of 16, then
// the rows' results into the last lane.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define FMD_MAX_DPP(ctrl, rows)                                                                    \
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, (ctrl), (rows), 0xf, false))
  FMD_MAX_DPP(0xB1, 0xf);    // lane ^ 1
  FMD_MAX_DPP(0x4E, 0xf);    // lane ^ 2
  FMD_MAX_DPP(0x141, 0xf);   // mirrored in 8
  FMD_MAX_DPP(0x140, 0xf);   // mirrored in 16
  FMD_MAX_DPP(0x142, 0xa);   // row 0 into 1, row 2 into 3
  FMD_MAX_DPP(0x143, 0xc);   // row 1 into 2 and 3
#undef FMD_MAX_DPP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t k) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)k, m);
    k = o > k ? o : k;
  }
  return k;
}
// Largest key of the work-group, in every thread.  turn alternates the words,
// so that one barrier per call is enough.
__device__ __forceinline__ uint64_t group_max(Shared& sh, uint64_t k, int turn) {
  k = wave_max_u64(k);
  if ((threadIdx.x & 63) == 0) sh.wave[turn & 1][threadIdx.x >> 6] = k;
  __syncthreads();
  uint64_t r = sh.wave[turn & 1][0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) r = sh.wave[turn & 1][i] > r ? sh.wave[turn & 1][i] : r;
  return r;
}
// How many of keys[0 .. n) are larger; eight reads in flight at a time.
__device__ __forceinline__ int larger(const uint64_t* keys, int n, uint64_t than) {
  int r = 0, i = 0;
  for (; i + 8 <= n; i += 8) {
    uint64_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = keys[i + j];
#pragma unroll
    for (int j = 0; j < 8; ++j) r += k[j] > than;
  }
  for (; i < n; ++i) r += keys[i] > than;
  return r;
}
__device__ __forceinline__ Stat group_join(Shared& sh, Stat a) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const Stat o = {__shfl_xor(a.m, m), __shfl_xor(a.s, m), __shfl_xor(a.t, m)};
    a = join(a, o);
  }
  if ((threadIdx.x & 63) == 0) sh.stat[threadIdx.x >> 6] = a;
  __syncthreads();
  a = sh.stat[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) a = join(a, sh.stat[i]);
  return a;
}

template <int DT> struct Elem;
template <> struct Elem<0> { typedef float T; };
template <> struct Elem<1> { typedef uint16_t T; };
template <> struct Elem<2> { typedef uint16_t T; };
template <int DT> __device__ __forceinline__ float widen(typename Elem<DT>::T v) {
  if constexpr (DT == 0) return v;
  else if constexpr (DT == 1) return f16_to_f32(v);
  else return bf16_to_f32(v);
}

// A lane's 16 values of a tile: VEC consecutive ones at VEC lane + 64 VEC k, as
// they lie in memory until they are used.  Rows need not start at 16-byte
// addresses (odd vocabularies): element alignment is said.
template <int DT> struct Raw {
  typedef typename Elem<DT>::T T;
  static constexpr int VEC = 16 / sizeof(T), N = kPer / VEC;
  typedef T V __attribute__((ext_vector_type(VEC)));
  typedef V U __attribute__((aligned(sizeof(T))));
  V v[N];
  static __device__ __forceinline__ int index(int e, int lane) {
    return (e / VEC) * (64 * VEC) + VEC * lane + e % VEC;
  }
  // past the row's end: the type's -inf
  static __device__ __forceinline__ T fill() {
    if constexpr (DT == 0) return -INFINITY;
    else return DT == 1 ? 0xfc00 : 0xff80;
  }
  __device__ __forceinline__ void load(const T* x, int at, int vocab, int lane) {
    if (at + kTile <= vocab) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = *(const U*)(x + at + index(k * VEC, lane));
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int i = at + index(k * VEC + j, lane);
          v[k][j] = i < vocab ? x[i] : fill();
        }
    }
  }
  __device__ __forceinline__ float get(int e) const { return widen<DT>(v[e / VEC][e % VEC]); }
};

// A tile's share of the lane's running statistics: v is used up.
__device__ __forceinline__ float add_tile(Stat& st, float* v) {
  // losers of round r lie at the odd multiples of 2^r, the winner at 0
#pragma unroll
  for (int r = 1; r < kPer; r <<= 1)
#pragma unroll
    for (int i = 0; i < kPer; i += 2 * r) {
      const float a = v[i], b = v[i + r];
      v[i] = top2(a, b);
      v[i + r] = low2(a, b);
    }
  const float tm = v[0], m = top2(st.m, tm), lo = low2(st.m, tm);
  const float mm = m == -INFINITY ? 0.f : m;
  // the tile's largest value against the running one: the smaller of them
  // loses, with all that was summed below it when that is the running one
  const float d = top2((lo - mm) * kLog2e, -1000.f), f = __builtin_amdgcn_exp2f(d);
  const bool grew = tm > st.m;
  const float n = grew ? st.s + 1.f : 1.f, u = grew ? st.t : 0.f;
  float s = f * n, t = f * (u + d * n);
  if (!grew) {
    s += st.s;
    t += st.t;
  }
  float ps = 0.f, pt = 0.f, err = 0.f;
  auto add = [&](float y) {
    y = top2(y, -1000.f);   // ruled out tokens: 2^-1000 is 0, and so is 0 * -1000
    const float p = __builtin_amdgcn_exp2f(y);
    ps += p;
    pt = fmaf(p, y, pt);
  };
  if (__any(!(fabsf(mm) <= kNear))) {
    // logits so large that r0 below would round by much, or not be finite
#pragma unroll
    for (int e = 1; e < kPer; ++e) add((v[e] - mm) * kLog2e);
  } else {
    // exponents are taken as v log2e - r0; r0's rounding, the same for all of
    // the tile, is put right in their sums
    const float r0 = mm * kLog2e;
    err = fmaf(mm, kLog2e, -r0);
#pragma unroll
    for (int e = 1; e < kPer; ++e) add(fmaf(v[e], kLog2e, -r0));
  }
  const float c = fmaf(-err, kLn2, 1.f);   // 2^-err
  st = {m, fmaf(c, ps, s), fmaf(c, pt - err * ps, t)};
  return tm;
}

// The wave's alternatives: lane i holds the i-th (0: none).
struct List {
  uint64_t mine;
  uint64_t last;   // of the top ones, in every lane
  __device__ __forceinline__ void insert(uint64_t k, int top, int lane) {
    const int at = __popcll(__ballot(mine > k));
    const uint64_t prev = __shfl_up((unsigned long long)mine, 1);
    mine = lane < at ? mine : lane == at ? k : prev;
    last = lane_u64(mine, top - 1);
  }
};

// A row's outputs from its joined parts (best in LDS, st in every thread).
__device__ __forceinline__ void finish(const LogprobArgs& a, const Shared& sh, Stat st, int row, float target) {
  // a row with +inf has no distribution, as one with a NaN (whose s is NaN)
  const float ls = st.m == INFINITY ? NAN : log1pf(st.s);
  const bool none = st.m == -INFINITY;   // every token ruled out: no distribution
  if (threadIdx.x == 0) {
    if (a.logp) a.logp[row] = target - st.m - ls;
    if (a.entropy) a.entropy[row] = none ? NAN : ls - kLn2 * st.t / (1.f + st.s);
  }
  for (int i = threadIdx.x; i < a.top; i += kThreads) {
    const uint64_t k = sh.joined[i];
    a.ids[(size_t)row * a.top + i] = (int32_t)key_index(k);
    a.best[(size_t)row * a.top + i] = key_value(k) - st.m - ls;
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_num_sgpr(96))) logprob_kernel(LogprobArgs a, int splits, int per) {
  __shared__ Shared sh;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x % splits, row = blockIdx.x / splits;
  const typename Elem<DT>::T* x = (const typename Elem<DT>::T*)a.x + (size_t)row * a.ld;
  const int tiles = (a.vocab + kTile - 1) / kTile;
  const int t0 = split * per + w, t1 = min((split + 1) * per, tiles);
  // the asked token's logit, long before it is used; an id outside the
  // vocabulary has no probability
  float target = NAN;
  if (a.logp && threadIdx.x == 0) {
    const int t = a.target[row];
    if (t >= 0 && t < a.vocab) target = widen<DT>(x[t]);
  }
  Stat st = {-INFINITY, 0.f, 0.f};
  List list = {0, 0};
  // The work-group's common bound: when each of n waves has k values at or above
  // x and n k >= top, nothing below x is among the row's top.  A wave tells its
  // k-th value (as the order's upper half); the bound is the least told.
  const int active = max(1, min(kWaves, t1 - split * per)), k_own = (a.top + active - 1) / active;
  uint32_t told = 0;
  float common = NAN;   // NaN: no bound yet
  auto look = [&]() {
    uint32_t b = ~0u;
    // one lane a wave's word; absent waves' words are never the least
    if (lane < kWaves) b = __hip_atomic_load(&sh.told[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    b = ~wave_max_u32(~b);
    common = b ? key_value((uint64_t)b << 32) : NAN;
  };
  // Candidates: values at or above the common bound, and above the wave's last one
  // of the tiles before (whose indices are lower: an equal later one loses); any,
  // NaN too, as long as there is no bound.
  auto collect = [&](const Raw<DT>& raw, int t, float tm) {
    const float own = list.last ? key_value(list.last) : NAN;
    auto open = [&](float f) { return !(f < common) & !(f <= own); };
    if (!__any(open(tm))) return;
    look();
    if (!__any(open(tm))) return;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float f = raw.get(e);
      uint64_t who = __ballot(open(f) & (t * kTile + Raw<DT>::index(e, lane) < a.vocab));
      while (who) {
        const int l = __ffsll((long long)who) - 1;
        who &= who - 1;
        const float fl = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), l));
        const uint64_t k = rank_key(fl, (uint32_t)(t * kTile + Raw<DT>::index(e, l)));
        if (k > list.last) list.insert(k, a.top, lane);
      }
    }
    const uint32_t now = (uint32_t)(lane_u64(list.mine, k_own - 1) >> 32);
    if (now > told) {
      told = now;
      if (lane == 0) __hip_atomic_store(&sh.told[w], now, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  };
  Raw<DT> next;
  auto take = [&](int t, Raw<DT>& raw) {
    raw = next;
    if (t + kWaves < t1) next.load(x, (t + kWaves) * kTile, a.vocab, lane);
    float v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = raw.get(e);
    return add_tile(st, v);
  };
  Raw<DT> raw;
  float tm = -INFINITY;
  if (t0 < t1) {
    next.load(x, t0 * kTile, a.vocab, lane);
    tm = take(t0, raw);
  }
  if (a.top > 0) {
    // what the waves can tell from their first tiles: the k-th largest of the
    // lanes' largest values
    uint32_t b = t0 < t1 ? (uint32_t)(rank_key(tm, 0) >> 32) : 0;
    for (int n = 0; n < k_own; ++n) {
      told = wave_max_u32(b);
      const uint64_t who = __ballot(b == told);
      if (lane == __ffsll((long long)who) - 1) b = 0;
    }
    if (lane == 0) sh.told[w] = t0 < t1 ? told : ~0u;
    __syncthreads();
    look();
    if (t0 < t1) collect(raw, t0, tm);
  }
  for (int t = t0 + kWaves; t < t1; t += kWaves) {
    tm = take(t, raw);
    if (a.top > 0) collect(raw, t, tm);
  }
  if (lane < a.top) sh.all[w * a.top + lane] = list.mine;
  st = group_join(sh, st);
  // group_join's barrier stands behind the lists, one after another.  Each of
  // their keys finds its place by counting the larger ones.
  const uint64_t key = threadIdx.x < kWaves * a.top ? sh.all[threadIdx.x] : 0;
  const int rank = larger(sh.all, kWaves * a.top, key);
  if (threadIdx.x < kMaxTop) sh.joined[threadIdx.x] = 0;
  __syncthreads();
  if (key && rank < a.top) sh.joined[rank] = key;
  __syncthreads();
  if (splits > 1) {
    // This piece's part, then a ticket: the work-group that draws a row's last
    // one finds all its parts written and joins them.  Parts are stored and
    // loaded past the XCDs' own L2s (agent scope), and a ticket is drawn once
    // the stores of its work-group have been answered, so no cache is written
    // back or dropped for them.  The last one leaves the tickets at 0 for the
    // next launch.
    uint32_t* const tickets = (uint32_t*)a.work;
    Part* const parts = (Part*)(tickets + 2 * kGroups) + (size_t)row * splits;
    if (threadIdx.x < a.top) put(&parts[split].keys[threadIdx.x], sh.joined[threadIdx.x]);
    if (threadIdx.x == 0) {
      put(&parts[split].ms, ((uint64_t)__builtin_bit_cast(uint32_t, st.s) << 32) | __builtin_bit_cast(uint32_t, st.m));
      put(&parts[split].t, (uint64_t)__builtin_bit_cast(uint32_t, st.t));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
      sh.ticket = __hip_atomic_fetch_add(tickets + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (sh.ticket != (uint32_t)splits - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(tickets + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int i = threadIdx.x;
    const int keys = splits * a.top;
    st = {-INFINITY, 0.f, 0.f};
    if (i < splits) {
      const uint64_t ms = get(&parts[i].ms);
      st = {__builtin_bit_cast(float, (uint32_t)ms), __builtin_bit_cast(float, (uint32_t)(ms >> 32)),
            __builtin_bit_cast(float, (uint32_t)get(&parts[i].t))};
    }
    if (keys <= kRanked) {
      // every key finds its place by counting the larger ones
      for (int k = i; k < keys; k += kThreads) sh.all[k] = get(&parts[k / a.top].keys[k % a.top]);
      if (i < kMaxTop) sh.joined[i] = 0;
      st = group_join(sh, st);   // its barrier stands behind the keys, too
      for (int k = i; k < keys; k += kThreads) {
        const uint64_t mine = sh.all[k];
        const int at = larger(sh.all, keys, mine);
        if (mine && at < a.top) sh.joined[at] = mine;
      }
    } else {
      // the parts' lists are in order: the largest of their heads, top times
      st = group_join(sh, st);
      int at = 0;
      uint64_t head = i < splits ? get(&parts[i].keys[0]) : 0;
      for (int n = 0; n < a.top; ++n) {
        const uint64_t k = group_max(sh, head, n);
        if (i == 0) sh.joined[n] = k;
        if (head == k && k) head = ++at < a.top ? get(&parts[i].keys[at]) : 0;
      }
    }
    __syncthreads();
  }
  finish(a, sh, st, row, target);
}

}  // namespace

// Pieces of a row: enough work-groups for the device, each wave a tile at least,
// and at most one piece per thread of the joining work-group.
static int logprob_splits(int rows, int vocab) {
  const int most = std::min((vocab + kWaves * kTile - 1) / (kWaves * kTile), kThreads);
  return std::min((kGroups + rows - 1) / rows, most);
}
int logprob_max_top() { return kMaxTop; }
// Rows in several pieces: fewer than kGroups of them, and fewer than 2 kGroups
// pieces.  One size for every call; the tickets come first.
size_t logprob_work_bytes() { return 2 * kGroups * (sizeof(uint32_t) + sizeof(Part)); }
size_t logprob_ticket_words() { return 2 * kGroups; }

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const int tiles = (a.vocab + kTile - 1) / kTile;
  int splits = logprob_splits(a.rows, a.vocab);
  const int per = ((tiles + splits - 1) / splits + kWaves - 1) / kWaves * kWaves;
  splits = (tiles + per - 1) / per;
  if (a.top > kMaxTop || (splits > 1 && (int64_t)a.rows * splits > 2 * kGroups)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)a.rows * splits), block(kThreads);
  if (a.dtype == 0) hipLaunchKernelGGL(logprob_kernel<0>, grid, block, 0, s, a, splits, per);
  else if (a.dtype == 1) hipLaunchKernelGGL(logprob_kernel<1>, grid, block, 0, s, a, splits, per);
  else hipLaunchKernelGGL(logprob_kernel<2>, grid, block, 0, s, a, splits, per);
  return hipGetLastError();
}
