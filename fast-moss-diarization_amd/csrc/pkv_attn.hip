// Attention over the paged 4-bit KV cache: causal, with an optional sliding
// window whose first tokens (the sinks) stay visible.
//
// A query at position p sees the keys j <= p with j > p - window or j < sinks
// (window 0: every j <= p), its own among them, so no row is empty.
//   ctx = sum_j softmax_j(q . k_j / sqrt(128)) v_j
// in one pass over the keys with a running maximum m and sum l; scores, m, l
// and the sums over v are 32 bits.
//
// One new token (a decode step) is bound by the cache's bytes, 136 per key and
// KV head.  A wave takes whole pages, by direct-to-LDS copies, the next page's in
// flight while this one is computed.
// - S^T = K q^T by 16x16x32 MFMAs: lane (c, g) = (l % 16, l / 16) of tile mt
//   holds row c of the A operand, which is token 16 (c/4) + 4 mt + c%4, and of
//   it the dims of block g, whose scale is then one per lane:
//   v_cvt_scalef32_pk turns two codes into two scaled 16-bit values, exactly.
//   The rows are picked so that a lane's 16 scores are tokens 16 g .. 16 g + 15.
// - The heads of a KV group fill 1, 2 or 4 of the MFMA's 16 columns; the others
//   carry what would otherwise take more instructions.  Column c is head c %
//   REP, block (c / REP) % 4 of V's dims and term c / (4 REP): each column's
//   p_j is multiplied by its V block's scale (the scale is along the sum's
//   tokens and so cannot be an operand's own), and its terms split that product
//   into bf16 parts, hi + lo, so that p keeps 16 bits where rounding to bf16
//   alone keeps 8 (32-bit activations: three terms, 24 bits).
// - O^T += V^T P^T with V's codes transposed by LDS 4-bit transpose reads (lane
//   = dim, 16 tokens in 8 bytes) and widened without a scale.
// A row's pages are cut into items so that a launch fills the device once (two
// work-groups on each CU, what its LDS holds of two pages a wave); the last of a
// row's items to end joins them.  16 rows of 8,000-40,000 keys, 440 MB: 75 us, 5.9
// TB/s.  8 rows of 4096, 36 MB: 11.0-12.4 us; cut for two rounds with K in
// registers and one page in flight it was 17.6.
//
// Many new tokens (prefill) are bound by the products and the softmax.  A
// work-group holds the queries of a tile, waves own (head, 16 QS positions);
// each page is widened once into 16-bit K and V blocks in LDS (double
// buffered, the next page's codes in registers meanwhile).  The pages of all
// tiles, one after another, are cut into equal runs for two work-groups on each
// CU; tiles that a cut goes through are joined by a second kernel.  8 x 512
// queries at 1,500-8,000: 207 us and 15 us for the join, 193 GFLOP at 0.87
// PFLOP/s; the matrix pipe is busy 38% of the time, VALU issue 47%, LDS 30%, and
// two waves on a SIMD overlap them only in part.  p is rounded to the 16-bit type
// once (l sums the rounded values).
// Measured on that case: one work-group of eight waves on a CU 258 us; reads
// right before their products (the compiler's order) +6%; pages and tables by
// generic pointers, whose returns LDS waits wait for, +9%; without the raised wave
// priority around the products +3%.
#include <algorithm>
#include <type_traits>

#include "fmd_common.h"
#include "fmd_kernels.h"

namespace {

constexpr int HD = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.f;   // log2 units that a row's scores may exceed its reference m by

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two codes (byte SEL of w) times the power of two sc, as 16-bit values.
template <bool F16, int SEL>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float sc) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, SEL));
}
template <bool F16>
__device__ __forceinline__ u32x4 widen8(uint32_t w, float sc) {
  return u32x4{widen2<F16, 0>(w, sc), widen2<F16, 1>(w, sc), widen2<F16, 2>(w, sc),
               widen2<F16, 3>(w, sc)};
}
template <bool F16>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ float rd_bf16(float v) { return rd<ACT_BF16>(v); }

// Eight activation values at p as NT bf16 (16-bit activations: one operand in
// their own type) terms that add up to them.
template <int A, int NT>
__device__ __forceinline__ void load_terms(const void* q, size_t at, bool ok, u32x4* t) {
  if constexpr (A != ACT_F32) {
    t[0] = ok ? *(const u32x4*)((const uint16_t*)q + at) : u32x4{0, 0, 0, 0};
  } else {
    f32x4 a[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (ok) {
      a[0] = *(const f32x4*)((const float*)q + at);
      a[1] = *(const f32x4*)((const float*)q + at + 4);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = a[i >> 1][2 * (i & 1)], y = a[i >> 1][2 * (i & 1) + 1];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        t[n][i] = pack2<false>(x, y);
        x -= rd_bf16(x);
        y -= rd_bf16(y);
      }
    }
  }
}

// Global memory by its address space: through a generic pointer the loads would
// be flat ones, which LDS waits wait for, too.
typedef const __attribute__((address_space(1))) uint8_t* gmem_t;
typedef const __attribute__((address_space(1))) u32x4* gmem16_t;

// The plan, which no kernel that reads it here writes: scalar loads.
typedef const __attribute__((address_space(4))) int32_t* plan_t;
__device__ __forceinline__ plan_t plan_of(const int32_t* p) { return (plan_t)(uint64_t)(uintptr_t)p; }
__device__ __forceinline__ gmem_t pool_of(plan_t plan) {
  return (gmem_t)(((uint64_t)(uint32_t)plan[PH_POOL + 1] << 32) | (uint32_t)plan[PH_POOL]);
}

// Words that one work-group leaves for another of the same launch.
__device__ __forceinline__ void put(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- one new token --------------------------------------------------------

constexpr int kDecWaves = 4;

template <int A, int REP>
__global__ void __launch_bounds__(64 * kDecWaves, 2) pkv_decode_kernel(PkvAttnArgs a) {
  constexpr bool F16 = A == ACT_F16;
  constexpr int NT = A == ACT_F32 ? 3 : 1;          // terms of q
  constexpr int PT = A == ACT_F32 ? 3 : 2;          // terms of p
  constexpr int TPP = 4 / REP;                      // terms that the columns of one MFMA hold
  constexpr int PASSES = (PT + TPP - 1) / TPP;
  constexpr int ESZ = A == ACT_F32 ? 4 : 2;
  constexpr int QB = REP * HD * ESZ;                // bytes of the group's queries
  constexpr int QC = (QB + 1023) / 1024;            // copies of 1 KiB for them
  constexpr int SLOT = kPkvHeadBytes;               // a page of one head
  constexpr int COPIES = 9;                         // copies of 1 KiB (the last of 512 B) for it
  // per wave: two pages and the queries, all by direct-to-LDS copies, so that the
  // only loads that are waited for are counted here
  __shared__ __attribute__((aligned(1024))) uint8_t sPage[kDecWaves][2 * SLOT + 1024 * QC];
  __shared__ float sM[kDecWaves][REP], sL[kDecWaves][REP];
  __shared__ uint32_t sTicket;
  float* const sO = (float*)&sPage[0][0];           // [wave][REP][HD], after the loop
  const plan_t plan = plan_of(a.plan);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int head = blockIdx.y, nh = a.nkv * REP;
  const int blk = (c / REP) & 3, term = c / (4 * REP);
  const float c2 = a.scale * kLog2e;
  const int n_items = plan[PH_NDEC];
  const size_t stride = (size_t)a.nkv * kPkvHeadBytes;       // bytes of a page
  const uint8_t* layer = (const uint8_t*)(uint64_t)(pool_of(plan) + (size_t)a.layer * plan[PH_PAGES] * stride +
                                                   (size_t)head * kPkvHeadBytes);
  uint8_t* const mine = &sPage[w][0];
  const uint32_t lds = lds_addr(mine);
  // Copy j < 4 brings the K codes of tokens 16 j .. 16 j + 15, j + 4 their V
  // codes.  Token t's 16-byte chunk x lies at chunk x ^ (t / 16) for K and x ^
  // ((t / 4) % 4) for V: the 16 tokens of a fragment read, and those of a
  // transpose read, then fall in distinct banks.
  uint32_t ksrc[4], vsrc;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    ksrc[j] = (uint32_t)((16 * j + (lane >> 2)) * 64 + (((lane & 3) ^ j) << 4));
  vsrc = (uint32_t)(kPkvV + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 4) & 3)) << 4));   // + 1024 j
  auto fetch = [&](int id, int slot) {
    const uint8_t* page = layer + (size_t)id * stride;
    const uint32_t to = lds + slot * SLOT;
#pragma unroll
    for (int j = 0; j < 4; ++j) lds_copy16(page, ksrc[j], to + j * 1024);
#pragma unroll
    for (int j = 0; j < 4; ++j) lds_copy16(page, vsrc + j * 1024, to + kPkvV + j * 1024);
    if (lane < 32) lds_copy16(page, (uint32_t)(kPkvKs + 16 * lane), to + kPkvKs);
  };

  for (int it = blockIdx.x; it < n_items; it += gridDim.x) {
    const plan_t ip = plan + PH_ITEMS + it * (int)(sizeof(PkvDecItem) / 4);
    PkvDecItem item;
    item.row = ip[0];
    item.pos = ip[1];
    item.table = ip[2];
    item.sp = ip[3];
    item.wp = ip[4];
    item.v0 = ip[5];
    item.v1 = ip[6];
    item.slot = ip[7];
    item.first = ip[8];
    item.parts = ip[9];
    if (item.row >= a.rows) continue;
    const plan_t table = plan + item.table;
    auto page_of = [&](int v) { return v < item.sp ? v : item.wp + (v - item.sp); };
    auto id_of = [&](int v) { return table[page_of(min(v, item.v1 - 1))]; };   // read a step ahead
    const int first = item.v0 + w;
    int id = ip[10 + w];
    {
      const uint8_t* q = (const uint8_t*)a.q + ((size_t)item.row * nh + head * REP) * (HD * ESZ);
#pragma unroll
      for (int j = 0; j < QC; ++j)
        if (j * 1024 + 16 * lane < QB) lds_copy16(q, (uint32_t)(j * 1024 + 16 * lane), lds + 2 * SLOT + j * 1024);
    }
    if (first < item.v1) fetch(id, 0);
    id = id_of(first + kDecWaves);
    f32x4 o[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m2 = -INFINITY, mr = 0.f, l = 0.f;   // mr: m2, or 0 while no key was seen
    u32x4 qf[4][NT];

    int slot = 0;
    for (int v = first; v < item.v1; v += kDecWaves, slot ^= 1) {
      // the next page's copies go out, this page's are waited for.  The slot they
      // go to was read in the step before: its reads have been answered, since
      // what they brought has been used.
      if (v + kDecWaves < item.v1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        fetch(id, slot ^ 1);
        id = id_of(v + 2 * kDecWaves);
        wait_vm<COPIES>();
      } else {
        wait_vm<0>();
      }
      asm volatile("" ::: "memory");
      if (v == first) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          load_terms<A, NT>(mine + 2 * SLOT, (size_t)(c % REP) * HD + 32 * g + 8 * j, true, qf[j]);
      }
      const uint8_t* page = mine + slot * SLOT;
      const int kb = page_of(v) * kPkvPage;
      const uint32_t ks = *(const uint32_t*)(page + kPkvKs + 4 * (16 * g + c));
      const u32x4 vs = *(const u32x4*)(page + kPkvVs + 64 * blk + 16 * g);
      f32x4 s[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const float sc = __builtin_bit_cast(float, ((ks >> (8 * mt)) & 0xffu) << 23);
        const u32x4 k = *(const u32x4*)(page + (16 * (c >> 2) + 4 * mt + (c & 3)) * 64 + ((g ^ (c >> 2)) << 4));
        s[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 kf = widen8<F16>(k[j], sc);
#pragma unroll
          for (int n = 0; n < NT; ++n) s[mt] = mfma<F16>(kf, qf[j][n], s[mt]);
        }
      }
      // tokens 16 g + 4 mt + i of the page
      const bool full = kb + kPkvPage - 1 <= item.pos &&
                        (a.window == 0 || kb > item.pos - a.window || kb + kPkvPage <= a.sinks);
      if (!full) {
        const int behind = a.window ? item.pos - a.window : -1;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = kb + 16 * g + e;
          const bool hidden = (j > item.pos) | ((j <= behind) & (j >= a.sinks));
          s[e >> 2][e & 3] = hidden ? -INFINITY : s[e >> 2][e & 3];
        }
      }
      float bm = s[0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) bm = fmaxf(bm, s[e >> 2][e & 3]);
      if (__any(fmaf(bm, c2, -mr) > kGrow || m2 == -INFINITY)) {
        bm = fmaxf(bm, __shfl_xor(bm, 16));
        bm = fmaxf(bm, __shfl_xor(bm, 32));
        const float mn = fmaxf(m2, bm * c2), nr = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m2 - nr);
        m2 = mn;
        mr = nr;
        l *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] *= f;
      }
      // p' = p * 2^(scale - 127): one exponential each, so that a masked
      // token's p' is 0 whatever its scale byte is
      float p[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = fmaf(s[e >> 2][e & 3], c2, -mr);
        l += __builtin_amdgcn_exp2f(x);
        const uint32_t byte = (vs[e >> 2] >> (8 * (e & 3))) & 0xffu;
        p[e] = __builtin_amdgcn_exp2f(x + ((float)byte - 127.f));
      }
      const uint8_t* vb = page + kPkvV;
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
      u32x4 pf[PASSES][2];
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float x = p[e], y = p[e + 1];
          // the column's term of the split: 0 the value, 1 what rounding left ..
          const int tt = ps * TPP + term;
#pragma unroll
          for (int n = 1; n < PT; ++n) {
            if (ps * TPP + TPP - 1 < n) break;   // no column of this pass has it
            const float rx = rd_bf16(x), ry = rd_bf16(y);
            if (tt >= n) {
              x -= rx;
              y -= ry;
            }
          }
          if ((ps + 1) * TPP > PT && tt >= PT) x = y = 0.f;
          pf[ps][e >> 3][(e & 7) >> 1] = pack2<false>(x, y);
        }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        // 16 tokens of dim 16 d + c: lane c of group g names token 16 g + c's
        // 8 bytes of dims 16 d ..
        const int t = 16 * g + c;
        const i32x2 vt = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (lds_i32x2*)(vb + t * 64 + (((d >> 1) ^ ((t >> 2) & 3)) << 4) + 8 * (d & 1)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 vf = widen8<false>((uint32_t)vt[h], 1.f);
#pragma unroll
          for (int ps = 0; ps < PASSES; ++ps) o[d] = mfma<false>(vf, pf[ps][h], o[d]);
        }
      }
    }
    wait_vm<0>();   // the queries of a wave without pages, too
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // the terms of a column add up; dims 32 b .. come from block b's columns
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = o[d][i];
        if constexpr (REP == 1) x += __shfl_xor(x, 4);
        if constexpr (REP <= 2) x += __shfl_xor(x, 8);
        o[d][i] = x;
      }
    __syncthreads();   // every wave has read its V codes
#pragma unroll
    for (int d = 0; d < 8; ++d)
      if (c < 4 * REP && blk == d >> 1)
        *(f32x4*)&sO[(w * REP + c % REP) * HD + 16 * d + 4 * g] = o[d];
    if (c < REP && g == 0) {
      sM[w][c] = m2;
      sL[w][c] = l;
    }
    __syncthreads();
    // (m, l, o) of the item's waves joined, REP * HD values over the threads
    constexpr int NV = (REP * HD + 64 * kDecWaves - 1) / (64 * kDecWaves);
    const bool whole = item.parts == 1;
    auto value = [&](int k) { return (int)threadIdx.x + k * 64 * kDecWaves; };
    auto store = [&](int i, float x, float L) {
      ((typename ActT<A>::T*)a.out)[((size_t)item.row * nh + head * REP) * HD + i] = st_act<A>(x / L);
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = value(k), r = i / HD;
      if (i >= REP * HD) break;
      float M = sM[0][r];
#pragma unroll
      for (int j = 1; j < kDecWaves; ++j) M = fmaxf(M, sM[j][r]);
      const float R = M == -INFINITY ? 0.f : M;
      float L = 0.f, x = 0.f;
#pragma unroll
      for (int j = 0; j < kDecWaves; ++j) {
        // a wave without pages has m = -inf, l = 0 and o = 0
        const float f = __builtin_amdgcn_exp2f(sM[j][r] - R);
        L += f * sL[j][r];
        x += f * sO[j * REP * HD + i];
      }
      if (whole) {
        store(i, x, L);
      } else {
        // past the XCD's own L2: the row's last item reads them
        const size_t u = ((size_t)item.slot * a.nkv + head) * REP;
        put(a.dec_o + u * HD + i, x);
        if (i % HD == 0) {
          put(a.dec_ml + 2 * (u + r), M);
          put(a.dec_ml + 2 * (u + r) + 1, L);
        }
      }
    }
    if (!whole) {
      // A ticket, drawn once this work-group's stores have been answered: the
      // last of a row's items finds all of them and joins them.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      uint32_t* const ticket = a.tickets + (size_t)item.first * a.nkv + head;
      if (threadIdx.x == 0) sTicket = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (sTicket == (uint32_t)item.parts - 1) {
        if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int i = value(k), r = i / HD;
          if (i >= REP * HD) break;
          auto unit = [&](int p) { return ((size_t)(item.first + p) * a.nkv + head) * REP; };
          // parts in blocks of eight, each with a running maximum: the loads of
          // a block are in flight together
          float M = -INFINITY, L = 0.f, x = 0.f;
          for (int p0 = 0; p0 < item.parts; p0 += 8) {
            float m8[8], l8[8], o8[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              const size_t u = unit(min(p0 + p, item.parts - 1));
              m8[p] = get(a.dec_ml + 2 * (u + r));
              l8[p] = get(a.dec_ml + 2 * (u + r) + 1);
              o8[p] = get(a.dec_o + u * HD + i);
            }
            float N = M;
#pragma unroll
            for (int p = 0; p < 8; ++p) N = fmaxf(N, m8[p]);
            const float R = N == -INFINITY ? 0.f : N, f0 = __builtin_amdgcn_exp2f(M - R);
            L *= f0;
            x *= f0;
            M = N;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              if (p0 + p >= item.parts) break;
              const float f = __builtin_amdgcn_exp2f(m8[p] - R);
              L += f * l8[p];
              x += f * o8[p];
            }
          }
          store(i, x, L);
        }
      }
    }
    __syncthreads();   // before the next item's copies overwrite sO
  }
}

// ---- many new tokens --------------------------------------------------------

// Waves of a work-group and sets of 16 positions of a wave.
template <int A, int REP> struct PreShape {
  static constexpr int QS = A == ACT_F32 ? 1 : 2;
  static constexpr int NW = 4;
  static constexpr int TP = 16 * QS * (NW / REP);   // positions of a tile
};

__device__ __forceinline__ int swk(int t) { return t & 15; }
__device__ __forceinline__ int swv(int t) { return (t & 7) << 1; }

template <int A, int REP>
__global__ void __launch_bounds__(64 * (PreShape<A, REP>::NW), 2) pkv_prefill_kernel(PkvAttnArgs a) {
  constexpr bool F16 = A == ACT_F16;
  constexpr int NT = A == ACT_F32 ? 3 : 1;     // terms of q and of p
  constexpr int QS = PreShape<A, REP>::QS, NW = PreShape<A, REP>::NW, TP = PreShape<A, REP>::TP;
  constexpr int NTH = 64 * NW, CH = 512 / NTH; // 16-byte chunks of codes per thread and page
  constexpr int BLK = kPkvPage * HD;
  __shared__ __attribute__((aligned(16))) uint16_t sK[2][BLK];
  __shared__ __attribute__((aligned(16))) uint16_t sV[2][BLK];
  const plan_t plan = plan_of(a.plan);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int qr = lane & 15, kg = lane >> 4;
  const int r = w % REP, half = w / REP, nh = a.nkv * REP;
  const float c2 = a.scale * kLog2e;
  const size_t stride = (size_t)a.nkv * kPkvHeadBytes;
  const int n_work = plan[PH_NWORK], n_units = n_work * a.nkv;
  const gmem_t pool = pool_of(plan) + (size_t)a.layer * plan[PH_PAGES] * stride;

  for (int un = blockIdx.x; un < n_units; un += gridDim.x) {
    // Neighbours of a KV head (a sequence's tiles) read the same pages: each XCD
    // (work-groups are dealt round-robin) takes a contiguous run.
    int unit = un;
    {
      const int per = n_units >> 3;
      if (un < 8 * per) unit = (un & 7) * per + (un >> 3);
    }
    const int head = unit / n_work;
    const plan_t work = plan + plan[PH_WORK] + unit % n_work;
    for (int it = work[0], end = work[1]; it < end; ++it) {
      const plan_t ip = plan + plan[PH_PITEM] + it * (int)(sizeof(PkvPreItem) / 4);
      PkvPreItem item;
      item.row = ip[0];
      item.pos = ip[1];
      item.n = ip[2];
      item.table = ip[3];
      item.sp = ip[4];
      item.wp = ip[5];
      item.v0 = ip[6];
      item.v1 = ip[7];
      item.slot = ip[8];
      const int rows = min(item.n, a.rows - item.row);
      if (rows <= 0) continue;
      const int h = head * REP + r;
      const plan_t table = plan + item.table;
      const gmem_t hbase = pool + (size_t)head * kPkvHeadBytes;
      auto page_of = [&](int v) { return v < item.sp ? v : item.wp + (v - item.sp); };
      const int last = item.pos + item.n - 1;      // the tile's last position

      int lim[QS], behind[QS];   // the last visible key, the last one behind the window
      u32x4 qf[QS][4][NT];
      float m2[QS], mr[QS];
      f32x4 o[QS][8], ls[QS];
#pragma unroll
      for (int qs = 0; qs < QS; ++qs) {
        const int my = 16 * (QS * half + qs) + qr;
        const bool ok = my < rows;
        lim[qs] = ok ? item.pos + my : item.pos;   // rows past the end see what the first does
        behind[qs] = a.window ? lim[qs] - a.window : -1;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          load_terms<A, NT>(a.q, ((size_t)(item.row + my) * nh + h) * HD + 32 * ks + 8 * kg, ok, qf[qs][ks]);
        m2[qs] = -INFINITY;
        mr[qs] = 0.f;
        ls[qs] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < 8; ++d) o[qs][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const uint32_t one2 = pack2<F16>(1.f, 1.f);
      const u32x4 ones = u32x4{one2, one2, one2, one2};

      // Codes of chunk x of a page (x < 256: K, else V): token (x / 4) % 64, block x % 4.
      u32x4 raw[CH];
      int rsc[CH];
      auto fetch = [&](int v) {
        const gmem_t hp = hbase + (size_t)table[page_of(v)] * stride;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int x = i * NTH + tid, t = (x >> 2) & 63, b = x & 3;
          raw[i] = *(gmem16_t)(hp + 16 * x);
          rsc[i] = hp[x < 256 ? kPkvKs + 64 * b + 4 * (4 * (t >> 4) + (t & 3)) + ((t >> 2) & 3)
                              : kPkvVs + 64 * b + t];
        }
      };
      // Widened into LDS.  K's NaN scale makes the token's scores NaN; V's values
      // are kept finite (they meet p = 0 of the rows that do not see the token),
      // and what lies past the last visible token, which no one may have
      // written, is 0.
      auto stage = [&](int v, int buf) {
        const int kb = page_of(v) * kPkvPage;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int x = i * NTH + tid, t = (x >> 2) & 63, b = x & 3;
          const bool isv = x >= 256;
          int byte = rsc[i];
          if (isv && byte == 255) byte = 127;
          const float sc = __builtin_bit_cast(float, (uint32_t)byte << 23);
          if (kb + t > last) raw[i] = u32x4{0, 0, 0, 0};
          uint16_t* row = (isv ? sV[buf] : sK[buf]) + t * HD;
          const int sw = isv ? swv(t) : swk(t);
#pragma unroll
          for (int j = 0; j < 4; ++j) *(u32x4*)(row + (((4 * b + j) ^ sw) << 3)) = widen8<F16>(raw[i][j], sc);
        }
      };
      fetch(item.v0);   // an item has a page at least
      stage(item.v0, 0);
      __syncthreads();
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      for (int v = item.v0, buf = 0; v < item.v1; ++v, buf ^= 1) {
        const int after = min(v + 1, item.v1 - 1);   // the last page once more, so that no branch is needed
        fetch(after);
        const int kb = page_of(v) * kPkvPage;
        const uint16_t* kbuf = sK[buf];
        const uint16_t* vbuf = sV[buf];
        // LDS reads go out a group ahead of the products that use them (a group is
        // 8 products, 128 cycles; a read takes about as long): K by tile, V by
        // half-block of tokens and half of the dims.  The scheduling barriers keep
        // the compiler from pulling them back together.
        f32x4 s[4][QS];
        u32x4 kf[2][4];
        auto read_k = [&](int mt) {
          const int t = 16 * mt + qr;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            kf[mt & 1][ks] = *(const u32x4*)(kbuf + t * HD + (((4 * ks + kg) ^ swk(t)) << 3));
        };
        s16x4 vf[2][4][2];
        auto read_v = [&](int gr) {
          const int t = 32 * (gr >> 1) + 4 * kg + (qr >> 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 4 * (gr & 1) + i;
            const uint16_t* at = vbuf + t * HD + (((2 * d + ((qr & 3) >> 1)) ^ swv(t)) << 3) + 4 * (qr & 1);
            vf[gr & 1][i][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
            vf[gr & 1][i][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * HD));
          }
        };
        read_k(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          if (mt < 3) read_k(mt + 1);
          else read_v(0);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int qs = 0; qs < QS; ++qs) s[mt][qs] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int qs = 0; qs < QS; ++qs)
#pragma unroll
              for (int n = 0; n < NT; ++n) s[mt][qs] = mfma<F16>(kf[mt & 1][ks], qf[qs][ks][n], s[mt][qs]);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const bool full = kb + kPkvPage - 1 <= item.pos &&
                          (a.window == 0 || kb > last - a.window || kb + kPkvPage <= a.sinks);
        bool grow = false;
        float bm[QS];
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
          if (!full) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int j = kb + 16 * (e >> 2) + 4 * kg + (e & 3);
              const bool hidden = (j > lim[qs]) | ((j <= behind[qs]) & (j >= a.sinks));
              s[e >> 2][qs][e & 3] = hidden ? -INFINITY : s[e >> 2][qs][e & 3];
            }
          }
          bm[qs] = s[0][qs][0];
#pragma unroll
          for (int e = 1; e < 16; ++e) bm[qs] = fmaxf(bm[qs], s[e >> 2][qs][e & 3]);
          grow |= fmaf(bm[qs], c2, -mr[qs]) > kGrow || m2[qs] == -INFINITY;
        }
        if (__any(grow)) {
#pragma unroll
          for (int qs = 0; qs < QS; ++qs) {
            float x = fmaxf(bm[qs], __shfl_xor(bm[qs], 16));
            x = fmaxf(x, __shfl_xor(x, 32));
            const float mn = fmaxf(m2[qs], x * c2), nr = mn == -INFINITY ? 0.f : mn;
            const float f = __builtin_amdgcn_exp2f(m2[qs] - nr);
            m2[qs] = mn;
            mr[qs] = nr;
            ls[qs] *= f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[qs][d] *= f;
          }
        }
        // O^T += V^T P^T over tokens 32 hb .. 32 hb + 31: k-slot i of group kg is
        // token 32 hb + 4 kg + i (i < 4) or 32 hb + 16 + 4 kg + i - 4, where S^T has them
        u32x4 pb[2][QS][NT];
        auto weigh = [&](int hb, int qs) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const f32x4 x = s[2 * hb + (e >> 2)][qs];
            float p0 = __builtin_amdgcn_exp2f(fmaf(x[e & 3], c2, -mr[qs]));
            float p1 = __builtin_amdgcn_exp2f(fmaf(x[(e & 3) + 1], c2, -mr[qs]));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              pb[hb][qs][n][e / 2] = pack2<F16>(p0, p1);
              if (n + 1 < NT) {
                p0 -= rd_bf16(p0);
                p1 -= rd_bf16(p1);
              }
            }
          }
        };
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) weigh(0, qs);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int gr = 0; gr < 4; ++gr) {
          const int hb = gr >> 1;
          if (gr < 3) read_v(gr + 1);
          __builtin_amdgcn_sched_barrier(0);
          if ((gr & 1) == 0) {
#pragma unroll
            for (int qs = 0; qs < QS; ++qs)
#pragma unroll
              for (int n = 0; n < NT; ++n) ls[qs] = mfma<F16>(ones, pb[hb][qs][n], ls[qs]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 4 * (gr & 1) + i;
            const u32x4 va = __builtin_bit_cast(
                u32x4, __builtin_shufflevector(vf[gr & 1][i][0], vf[gr & 1][i][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int qs = 0; qs < QS; ++qs)
#pragma unroll
              for (int n = 0; n < NT; ++n) o[qs][d] = mfma<F16>(va, pb[hb][qs][n], o[qs][d]);
          }
          // the second half's exponentials between the first half's products
          if (gr < 2 && gr < QS) weigh(1, gr);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        stage(after, buf ^ 1);
        __syncthreads();
      }
#pragma unroll
      for (int qs = 0; qs < QS; ++qs) {
        const int my = 16 * (QS * half + qs) + qr;
        if (my >= rows) continue;
        if (item.slot < 0) {
          const float inv = 1.f / ls[qs][0];
          const size_t at = ((size_t)(item.row + my) * nh + h) * HD + 4 * kg;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const f32x4 x = o[qs][d] * inv;
            if constexpr (A == ACT_F32) {
              *(f32x4*)((float*)a.out + at + 16 * d) = x;
            } else {
              uint32_t* p = (uint32_t*)((uint16_t*)a.out + at + 16 * d);
              p[0] = pack2<F16>(x[0], x[1]);
              p[1] = pack2<F16>(x[2], x[3]);
            }
          }
        } else {
          const size_t u = ((size_t)item.slot * a.nkv + head) * (TP * REP) + my * REP + r;
#pragma unroll
          for (int d = 0; d < 8; ++d) *(f32x4*)(a.pre_o + u * HD + 16 * d + 4 * kg) = o[qs][d];
          if (kg == 0) {
            a.pre_ml[2 * u] = m2[qs];
            a.pre_ml[2 * u + 1] = ls[qs][0];
          }
        }
      }
      __syncthreads();
    }
  }
}

// Joins the items of the tiles that were cut: a work-group per (8 query rows,
// KV head), 32 lanes and 4 dims each to a row.
template <int A, int REP>
__global__ void __launch_bounds__(256) pkv_prefill_join_kernel(PkvAttnArgs a) {
  constexpr int TR = PreShape<A, REP>::TP * REP, GR = TR / 8;
  const int32_t* plan = a.plan;
  const int head = blockIdx.y;
  for (int b = blockIdx.x; b < plan[PH_NSPLIT] * GR; b += gridDim.x) {
    const PkvSplit t = ((const PkvSplit*)(plan + plan[PH_SPLIT]))[b / GR];
    const int my = (b % GR) * 8 + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
    const int pos = my / REP, r = my % REP;
    if (pos >= min(t.n, a.rows - t.row)) continue;
    auto unit = [&](int i) { return ((size_t)(t.first + i) * a.nkv + head) * TR + my; };
    float M = -INFINITY;
    for (int i = 0; i < t.parts; ++i) M = fmaxf(M, a.pre_ml[2 * unit(i)]);
    const float R = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < t.parts; ++i) {
      const size_t u = unit(i);
      const float f = __builtin_amdgcn_exp2f(a.pre_ml[2 * u] - R);
      L += f * a.pre_ml[2 * u + 1];
      const f32x4 y = *(const f32x4*)(a.pre_o + u * HD + d);
      // an item that a row sees nothing of has l = 0 and o = 0
      x += y * f;
    }
    x *= 1.f / L;
    const size_t at = ((size_t)(t.row + pos) * a.nkv * REP + head * REP + r) * HD + d;
    if constexpr (A == ACT_F32) {
      *(f32x4*)((float*)a.out + at) = x;
    } else {
      uint32_t* p = (uint32_t*)((uint16_t*)a.out + at);
      p[0] = pack2<A == ACT_F16>(x[0], x[1]);
      p[1] = pack2<A == ACT_F16>(x[2], x[3]);
    }
  }
}

template <int A, int REP>
hipError_t launch_rep(const PkvAttnArgs& a, hipStream_t s) {
  if (a.ndec > 0)
    hipLaunchKernelGGL((pkv_decode_kernel<A, REP>), dim3(a.ndec, a.nkv), dim3(64 * kDecWaves), 0, s, a);
  if (a.nwork > 0) {
    hipLaunchKernelGGL((pkv_prefill_kernel<A, REP>), dim3(a.nwork * a.nkv),
                       dim3(64 * PreShape<A, REP>::NW), 0, s, a);
    if (a.nsplit > 0 || a.captured)
      hipLaunchKernelGGL((pkv_prefill_join_kernel<A, REP>),
                         dim3(std::max(a.nsplit, 1) * (PreShape<A, REP>::TP * REP / 8), a.nkv), dim3(256),
                         0, s, a);
  }
  return hipGetLastError();
}
template <int A>
hipError_t launch_act(const PkvAttnArgs& a, hipStream_t s) {
  switch (a.rep) {
    case 1: return launch_rep<A, 1>(a, s);
    case 2: return launch_rep<A, 2>(a, s);
    case 4: return launch_rep<A, 4>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_pkv_attn(int act, const PkvAttnArgs& a, hipStream_t s) {
  if (act == ACT_F32) return launch_act<ACT_F32>(a, s);
  if (act == ACT_F16) return launch_act<ACT_F16>(a, s);
  return launch_act<ACT_BF16>(a, s);
}

int pkv_tile_positions(int act, int rep) {
  auto of = [&](auto tag) {
    constexpr int A = decltype(tag)::value;
    return rep == 1 ? PreShape<A, 1>::TP : rep == 2 ? PreShape<A, 2>::TP : PreShape<A, 4>::TP;
  };
  return act == ACT_F32 ? of(std::integral_constant<int, ACT_F32>())
                        : of(std::integral_constant<int, ACT_BF16>());
}
