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
// Bound by one read of the logits.  A work-group takes a run of tiles of 4096
// values of one row, 16 in each thread's registers: the thread's running (M, S,
// T) needs one exponential per value, and only a tile whose largest value
// exceeds the row's current last alternative is searched for alternatives
// (largest first, a reduction over the work-group each), which after the first
// tiles is rare.  Rows are cut so that a launch has about kGroups work-groups;
// a second kernel joins a row's pieces.
//
// Alternatives are ordered by value, equal ones by index (lower first, -0 and 0
// are equal), NaN below -inf.
#include "fmd_common.h"
#include "fmd_kernels.h"

namespace {

constexpr int kThreads = 256, kPer = 16, kTile = kThreads * kPer;
constexpr int kGroups = 1024;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

struct Stat {
  float m, s, t;
};
__device__ __forceinline__ float expn(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

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
  const float d = b.m - a.m, f = expn(d), n = b.s + 1.f;
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

struct Shared {
  uint64_t best[kMaxTop];        // the row's alternatives so far, in order, 0: none
  uint64_t found[kMaxTop];       // a tile's
  uint64_t wave[2][kThreads / 64];
  Stat stat[kThreads / 64];
};

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
  for (int i = 1; i < kThreads / 64; ++i) r = sh.wave[turn & 1][i] > r ? sh.wave[turn & 1][i] : r;
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
  for (int i = 1; i < kThreads / 64; ++i) a = join(a, sh.stat[i]);
  return a;
}

// best := the first `top` of best and found (both in order).  One wave.
__device__ __forceinline__ void merge_lists(Shared& sh, int top, int n) {
  __syncthreads();
  const int i = threadIdx.x;
  uint64_t mine = 0;
  int rank = top;
  if (i < 2 * kMaxTop) {
    const bool old = i < kMaxTop;
    const int at = old ? i : i - kMaxTop;
    mine = old ? (at < top ? sh.best[at] : 0) : (at < n ? sh.found[at] : 0);
    if (mine) {
      rank = at;   // the keys before it in its own list, and the larger ones of the other
      const uint64_t* other = old ? sh.found : sh.best;
      const int m = old ? n : top;
      for (int j = 0; j < m; ++j) rank += other[j] > mine;
    }
  }
  __syncthreads();
  if (mine && rank < top) sh.best[rank] = mine;
  __syncthreads();
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

// 16 values of a tile: VEC consecutive ones at VEC tid + 256 VEC k.  Rows need
// not start at 16-byte addresses (odd vocabularies): element alignment is said.
template <int DT> struct Load {
  typedef typename Elem<DT>::T T;
  static constexpr int VEC = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(VEC)));
  typedef V U __attribute__((aligned(sizeof(T))));
  static __device__ __forceinline__ int index(int e) {
    return (e / VEC) * (kThreads * VEC) + VEC * threadIdx.x + e % VEC;
  }
  static __device__ __forceinline__ void tile(const T* x, int at, int vocab, float* o) {
#pragma unroll
    for (int k = 0; k < kPer / VEC; ++k) {
      const int i = at + index(k * VEC);
      if (i + VEC <= vocab) {
        const V v = *(const U*)(x + i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[k * VEC + j] = widen<DT>(v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[k * VEC + j] = i + j < vocab ? widen<DT>(x[i + j]) : -INFINITY;
      }
    }
  }
};

// A row's outputs from its joined parts (best in LDS, st in every thread).
template <int DT>
__device__ __forceinline__ void finish(const LogprobArgs& a, const Shared& sh, Stat st, int row) {
  // a row with +inf has no distribution, as one with a NaN (whose s is NaN)
  const float ls = st.m == INFINITY ? NAN : log1pf(st.s);
  const bool none = st.m == -INFINITY;   // every token ruled out: no distribution
  if (threadIdx.x == 0) {
    if (a.logp) {
      const int t = a.target[row];
      const typename Elem<DT>::T* x = (const typename Elem<DT>::T*)a.x + (size_t)row * a.ld;
      // an id outside the vocabulary has no probability
      a.logp[row] = t >= 0 && t < a.vocab ? widen<DT>(x[t]) - st.m - ls : NAN;
    }
    if (a.entropy) a.entropy[row] = none ? NAN : ls - st.t / (1.f + st.s);
  }
  for (int i = threadIdx.x; i < a.top; i += kThreads) {
    const uint64_t k = sh.best[i];
    a.ids[(size_t)row * a.top + i] = (int32_t)key_index(k);
    a.best[(size_t)row * a.top + i] = key_value(k) - st.m - ls;
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) logprob_kernel(LogprobArgs a, int splits, int per) {
  __shared__ Shared sh;
  const int split = blockIdx.x % splits, row = blockIdx.x / splits;
  const typename Elem<DT>::T* x = (const typename Elem<DT>::T*)a.x + (size_t)row * a.ld;
  const int tiles = (a.vocab + kTile - 1) / kTile;
  const int t0 = split * per, t1 = min(t0 + per, tiles);
  for (int i = threadIdx.x; i < kMaxTop; i += kThreads) sh.best[i] = 0;
  __syncthreads();
  Stat st = {-INFINITY, 0.f, 0.f};
  uint64_t floor_key = 0;   // the row's last alternative so far
  int turn = 0;
  for (int t = t0; t < t1; ++t) {
    float v[kPer];
    Load<DT>::tile(x, t * kTile, a.vocab, v);
    float tm = v[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) tm = fmaxf(tm, v[e]);
    const float m = fmaxf(st.m, tm);
    if (m != -INFINITY) {
      bool skip = tm > st.m;   // this tile's largest value leaves its own 1 out
      if (skip && st.m != -INFINITY) {
        const float d = st.m - m, f = expn(d), n = st.s + 1.f;
        st.t = f * (st.t + d * n);
        st.s = f * n;
      }
      st.m = m;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float d = v[e] - m;
        const bool self = skip && v[e] == m;
        skip = skip && !self;
        // d = -inf: e^d d is 0, not 0 * inf
        const float p = self ? 0.f : expn(d);
        st.s += p;
        st.t += v[e] == -INFINITY ? 0.f : p * d;
      }
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (v[e] != v[e]) st.s = NAN;   // also where every other value is -inf
    if (a.top == 0) continue;
    // Alternatives of this tile: its keys in falling order while they are
    // above the list's last.
    uint64_t mine = 0;
    auto refresh = [&](uint64_t below) {
      mine = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = t * kTile + Load<DT>::index(e);
        const uint64_t k = i < a.vocab ? rank_key(v[e], (uint32_t)i) : 0;
        mine = k < below && k > mine ? k : mine;
      }
    };
    const bool look = floor_key == 0 || !(tm <= key_value(floor_key));
    if (__syncthreads_or(look)) {
      if (look) refresh(~0ull);
      int n = 0;
      for (; n < a.top; ++n) {
        const uint64_t k = group_max(sh, mine, turn++);
        if (k <= floor_key) break;
        if (threadIdx.x == 0) sh.found[n] = k;
        if (mine == k) refresh(k);
      }
      if (n) {
        merge_lists(sh, a.top, n);
        floor_key = sh.best[a.top - 1];
      }
    }
  }
  st = group_join(sh, st);
  if (splits == 1) {
    finish<DT>(a, sh, st, row);
    return;
  }
  const size_t part = (size_t)row * splits + split;
  uint64_t* const keys = (uint64_t*)a.work + part * (kMaxTop + 2);
  for (int i = threadIdx.x; i < a.top; i += kThreads) keys[i] = sh.best[i];
  if (threadIdx.x == 0) *(Stat*)(keys + kMaxTop) = st;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) logprob_join_kernel(LogprobArgs a, int splits) {
  __shared__ Shared sh;
  const int row = blockIdx.x, i = threadIdx.x;
  const uint64_t* keys = (const uint64_t*)a.work + ((size_t)row * splits + i) * (kMaxTop + 2);
  Stat st = {-INFINITY, 0.f, 0.f};
  if (i < splits) st = *(const Stat*)(keys + kMaxTop);
  st = group_join(sh, st);
  // the pieces' lists are in order: the largest of their heads, top times
  int at = 0;
  uint64_t head = i < splits && a.top > 0 ? keys[0] : 0;
  for (int n = 0; n < a.top; ++n) {
    const uint64_t k = group_max(sh, head, n);
    if (i == 0) sh.best[n] = k;
    if (head == k && k) head = ++at < a.top ? keys[at] : 0;
  }
  __syncthreads();
  finish<DT>(a, sh, st, row);
}

}  // namespace

// Pieces of a row: enough work-groups for the device, at least a tile each and
// at most one per thread of the joining work-group.
static int logprob_splits(int rows, int vocab) {
  const int tiles = (vocab + kTile - 1) / kTile;
  const int want = (kGroups + rows - 1) / rows;
  return want < tiles ? (want > kThreads ? kThreads : want) : (tiles > kThreads ? kThreads : tiles);
}
int logprob_max_top() { return kMaxTop; }
// The largest launch that is cut (a row in more than one piece) has fewer than
// 2 kGroups pieces.
size_t logprob_work_bytes() { return (size_t)2 * kGroups * (kMaxTop + 2) * 8; }

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const int tiles = (a.vocab + kTile - 1) / kTile;
  int splits = logprob_splits(a.rows, a.vocab);
  const int per = (tiles + splits - 1) / splits;
  splits = (tiles + per - 1) / per;
  if (a.top > kMaxTop || (splits > 1 && (int64_t)a.rows * splits > 2 * kGroups)) return hipErrorInvalidValue;
#define FMD_LP(DT)                                                                                  \
  do {                                                                                              \
    hipLaunchKernelGGL(logprob_kernel<DT>, dim3((unsigned)a.rows * splits), dim3(kThreads), 0, s, a, \
                       splits, per);                                                                \
    if (splits > 1)                                                                                 \
      hipLaunchKernelGGL(logprob_join_kernel<DT>, dim3(a.rows), dim3(kThreads), 0, s, a, splits);   \
  } while (0)
  if (a.dtype == 0) FMD_LP(0);
  else if (a.dtype == 1) FMD_LP(1);
  else FMD_LP(2);
#undef FMD_LP
  return hipGetLastError();
}
