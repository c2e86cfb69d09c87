// Rows into and out of the paged 4-bit KV cache, and page copies.
//
// Append (Attention::forward's q/k norm, RoPE and cache append,
// qwen3.rs:213-241, into 4-bit pages): with x a head's 128 values, g the gain,
//   y = x / sqrt(mean(x^2) + eps) * g
//   z[i] = y[i] cos[i] - y[i + 64] sin[i],  z[i + 64] = y[i + 64] cos[i] + y[i] sin[i]
// q is z rounded once to the activation dtype; K is z and V the projection as
// 32-bit values, held as blocks of 32 dims b: 2^e c[d], e the smallest integer
// with max|b| <= 7 * 2^e and c the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties
// to the even code).  7 keeps every error within half a step of the widest
// gap (6 would spend a bit of scale on maxima in (6, 7], 8 clips them by up to
// a quarter); relative rms error of N(0, 1) blocks at 6 | 6.5 | 7 | 7.5 | 8:
// .1155 | .1131 | .1119 | .1120 | .1151.
//
// K is computed to 64 bits and rounded to 32: which code a value next to a border
// gets then does not depend on the order of the mean's sum.  q takes 32 bits.
//
// Bound by memory: 12,288 rows of 16 + 8 + 8 heads in bf16 are 151 MB of rows and
// 13 MB of pages, 30.6-32.4 us (5.0-5.3 TB/s, a device copy's rate).  Lanes of 16
// exchange by DPP and K's products stay in 32 bits where they are exact; with LDS
// exchanges and every product in 64 bits the same rows took 42 us.  Eight rows:
// 2.4-3.2 us, the chain plan -> tables -> pages.
//
// A token whose K or V of a head holds an infinity or a NaN gets scale 255 in
// all eight blocks of that head: it reads back as NaN, and so does every
// context that sees it.
#include "fmd_common.h"
#include "fmd_kernels.h"

namespace {

constexpr int HD = 128;

// Lowest and highest block exponent: what a cache returns is a value of the
// activation dtype (f16: 0.5 * 2^-23 is its smallest subnormal, 6 * 2^13 below
// its largest value; 32-bit and bf16 caches end where sums over a cache of
// 65,536 tokens still stay far inside 32 bits).
template <int A> constexpr int kLo = A == ACT_F16 ? -23 : -64;
template <int A> constexpr int kHi = A == ACT_F16 ? 13 : 64;

typedef const __attribute__((address_space(4))) int32_t* plan_t;   // scalar loads
typedef __attribute__((address_space(1))) uint8_t* gmem_t;         // no flat ones
typedef __attribute__((address_space(1))) uint32_t* gmem4_t;

// Where a row's token lies: its position, and the page.
struct Place {
  int pos;
  gmem_t page;
};
__device__ __forceinline__ Place place_of(const PkvRowArgs& a, plan_t plan, int rows, int row) {
  const plan_t at = (rows <= kPkvDirect ? plan + PH_WORDS : (plan_t)(uint64_t)a.far) + 2 * row;
  const uint64_t pool = ((uint64_t)(uint32_t)plan[PH_POOL + 1] << 32) | (uint32_t)plan[PH_POOL];
  Place p;
  p.pos = at[0];
  p.page = (gmem_t)pool + ((size_t)a.layer * plan[PH_PAGES] + at[1]) * a.nkv * (size_t)kPkvHeadBytes;
  return p;
}

__device__ __forceinline__ int kscale_at(int t, int blk) {
  return 64 * blk + 4 * (4 * (t >> 4) + (t & 3)) + ((t >> 2) & 3);
}

template <int A>
__device__ __forceinline__ void load8(const void* p, size_t at, float* o) {
  if constexpr (A == ACT_F32) {
    const f32x4 a = *(const f32x4*)((const float*)p + at), b = *(const f32x4*)((const float*)p + at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a[i];
      o[4 + i] = b[i];
    }
  } else {
    unpack8<A>(*(const u32x4*)((const uint16_t*)p + at), o);
  }
}
template <int A>
__device__ __forceinline__ void store8(void* p, size_t at, const float* v) {
  if constexpr (A == ACT_F32) {
    *(f32x4*)((float*)p + at) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)p + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)st_act<A>(v[2 * i]) | ((uint32_t)st_act<A>(v[2 * i + 1]) << 16);
    *(u32x4*)((uint16_t*)p + at) = w;
  }
}

// Largest magnitude of the 32 dims that a quad of lanes holds, as bits
// (magnitudes order like their bits, NaN above infinity).
__device__ __forceinline__ uint32_t quad_max_bits(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));
  return m;
}
// Scale byte of a block whose largest magnitude has bits m: the float exponent
// of m / 4, one more when the mantissa is above 1.75.
template <int A>
__device__ __forceinline__ int scale_byte(uint32_t m) {
  const int e = (int)((m + 0x1fffffu) >> 23) - 2;
  return min(max(e, 127 + kLo<A>), 127 + kHi<A>);
}
// Eight codes: v_cvt_scalef32_pk_fp4_f32 divides by the scale's power of two,
// rounds to nearest even and saturates at 6.
__device__ __forceinline__ uint32_t codes8(const float* x, int byte) {
  const float sc = __builtin_bit_cast(float, (uint32_t)byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], sc, 3);
  return w;
}

// K (k) and V (v) of one token and head, 8 dims per lane of a 16-lane row.
template <int A>
__device__ __forceinline__ void store_kv(gmem_t head, int t, int dc, const float* k, const float* v) {
  const uint32_t mk = quad_max_bits(k), mv = quad_max_bits(v);
  // any block of the row not finite: __ballot, then this row's 16 bits
  const uint64_t bad = __ballot(mk >= 0x7f800000u || mv >= 0x7f800000u);
  const bool nan = (bad >> (threadIdx.x & 48)) & 0xffffu;
  const int bk = scale_byte<A>(mk), bv = scale_byte<A>(mv);
  *(gmem4_t)(head + t * 64 + dc * 4) = nan ? 0u : codes8(k, bk);
  *(gmem4_t)(head + kPkvV + t * 64 + dc * 4) = nan ? 0u : codes8(v, bv);
  if ((dc & 3) == 0) {
    head[kPkvKs + kscale_at(t, dc >> 2)] = (uint8_t)(nan ? 255 : bk);
    head[kPkvVs + 64 * (dc >> 2) + t] = (uint8_t)(nan ? 255 : bv);
  }
}

// The value of lane ^ 8 of the 16-lane row: dims 64 on.
__device__ __forceinline__ float across(float v) { return FMD_DPP(v, 0x128); }

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// Norm and rotation of a q head's 8 dims 8 dc .., in 32 bits.
__device__ __forceinline__ void norm_rope_q(const float* x, const float* g, const float* c,
                                            const float* s, int dc, float eps, float* z) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
  ss = row16_sum(ss);
  const float r = __builtin_amdgcn_rsqf(ss * (1.f / HD) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = x[i] * r * g[i], o = across(y);
    z[i] = fmaf(y, c[i], dc < 8 ? -o * s[i] : o * s[i]);
  }
}

// The same of a K head as if in 64 bits.  What is exact in 32 bits is done
// there: a product of two 16-bit values, and of three bf16 ones (24 bits).
template <int A>
__device__ __forceinline__ void norm_rope_k(const float* x, const float* g, const float* c,
                                            const float* s, int dc, float eps, float* z) {
  double ss = 0.;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fma((double)x[i], (double)x[i], ss);
  ss += dpp64<0xB1>(ss);
  ss += dpp64<0x4E>(ss);
  ss += dpp64<0x141>(ss);
  ss += dpp64<0x140>(ss);
  // 1 / sqrt(m): the instruction's value, good to 2^-22 at least, and two Newton
  // steps, each of which squares its error
  const double m = fma(ss, 1. / HD, (double)eps);
  double r = __builtin_amdgcn_rsq(m);
#pragma unroll
  for (int k = 0; k < 2; ++k) r = fma(r, fma(-0.5 * m * r, r, 0.5), r);
  const bool lo = dc < 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float xo = across(x[i]), go = across(g[i]);
    double a, b;
    if constexpr (A == ACT_BF16) {
      a = (double)(x[i] * (g[i] * c[i]));
      b = (double)(xo * (go * s[i]));
    } else if constexpr (A == ACT_F16) {
      a = (double)x[i] * (double)(g[i] * c[i]);
      b = (double)xo * (double)(go * s[i]);
    } else {
      a = (double)x[i] * ((double)g[i] * (double)c[i]);
      b = (double)xo * ((double)go * (double)s[i]);
    }
    z[i] = (float)(r * (lo ? a - b : a + b));
  }
}

// One work-group per row, 16 lanes per head: nh q heads, then nkv lane rows
// that each take a head's K and V.
template <int A>
__global__ void pkv_append_kernel(PkvRowArgs a) {
  const plan_t plan = (plan_t)(uint64_t)a.plan;
  const int row = blockIdx.x, rows = plan[PH_ROWS];
  const int u = threadIdx.x >> 4, dc = threadIdx.x & 15;
  if (u >= a.nh + a.nkv) return;     // whole 16-lane rows: the shuffles below stay inside one
  // what the row index alone leads to, before the plan is looked at
  const size_t base = (size_t)row * (a.nh + 2 * a.nkv) * HD + 8 * dc;
  float x[8], v[8], g[8], c[8], sn[8], z[8];
  load8<A>(a.x, base + (size_t)u * HD, x);
  if (u >= a.nh) load8<A>(a.x, base + (size_t)(u + a.nkv) * HD, v);
  load8<A>(u < a.nh ? a.qn_w : a.kn_w, 8 * dc, g);
  if (row >= rows) return;
  const Place p = place_of(a, plan, rows, row);
  load8<A>(a.cos, (size_t)p.pos * (HD / 2) + 8 * (dc & 7), c);
  load8<A>(a.sin, (size_t)p.pos * (HD / 2) + 8 * (dc & 7), sn);
  if (u < a.nh) {
    norm_rope_q(x, g, c, sn, dc, a.eps, z);
    store8<A>(a.q_out, ((size_t)row * a.nh + u) * HD + 8 * dc, z);
  } else {
    norm_rope_k<A>(x, g, c, sn, dc, a.eps, z);
    store_kv<A>(p.page + (u - a.nh) * kPkvHeadBytes, p.pos % kPkvPage, dc, z, v);
  }
}

// The decoder's own tables hold the host's 32-bit cosines, of which one in some
// thousand is off by its last bit, and one in a million still is after the
// rounding to bf16.  A bit of a table moves the keys that lie next to a 4-bit
// border, by a quarter of their value: the append has tables of its own, from
// 64-bit cosines of the same angles.
template <int A>
__global__ void __launch_bounds__(256) pkv_rope_kernel(RopeFreqs f, int positions, void* cos_out, void* sin_out) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)positions * (HD / 2)) return;
  const double angle = (double)((float)(i / (HD / 2)) * f.inv[i % (HD / 2)]);
  // the empty asm keeps the two roundings apart: the compiler makes one of them
  float c = (float)cos(angle), s = (float)sin(angle);
  asm volatile("" : "+v"(c), "+v"(s));
  ((typename ActT<A>::T*)cos_out)[i] = st_act<A>(c);
  ((typename ActT<A>::T*)sin_out)[i] = st_act<A>(s);
}

// K and V rows as they are (already rotated) into the plan's positions.
template <int A>
__global__ void pkv_write_kernel(PkvRowArgs a) {
  const plan_t plan = (plan_t)(uint64_t)a.plan;
  const int row = blockIdx.x, rows = plan[PH_ROWS];
  const int u = threadIdx.x >> 4, dc = threadIdx.x & 15;
  if (u >= a.nkv) return;
  const size_t at = ((size_t)row * a.nkv + u) * HD + 8 * dc;
  float k[8], v[8];
  load8<A>(a.x, at, k);
  load8<A>(a.v, at, v);
  if (row >= rows) return;
  const Place p = place_of(a, plan, rows, row);
  store_kv<A>(p.page + u * kPkvHeadBytes, p.pos % kPkvPage, dc, k, v);
}

__device__ __forceinline__ void decode8(uint32_t w, int byte, float* o) {
  const float sc = __builtin_bit_cast(float, (uint32_t)byte << 23);   // 255: every value NaN
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
  o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
  o[4] = c[0]; o[5] = c[1]; o[6] = d[0]; o[7] = d[1];
}

// The plan's rows back, as the values they stand for.
template <int A>
__global__ void pkv_read_kernel(PkvRowArgs a) {
  const plan_t plan = (plan_t)(uint64_t)a.plan;
  const int row = blockIdx.x, rows = plan[PH_ROWS];
  if (row >= rows) return;
  const int u = threadIdx.x >> 4, dc = threadIdx.x & 15;
  if (u >= a.nkv) return;
  const Place p = place_of(a, plan, rows, row);
  const int t = p.pos % kPkvPage;
  const gmem_t head = p.page + u * kPkvHeadBytes;
  float k[8], v[8];
  decode8(*(gmem4_t)(head + t * 64 + dc * 4), head[kPkvKs + kscale_at(t, dc >> 2)], k);
  decode8(*(gmem4_t)(head + kPkvV + t * 64 + dc * 4), head[kPkvVs + 64 * (dc >> 2) + t], v);
  const size_t at = ((size_t)row * a.nkv + u) * HD + 8 * dc;
  if (a.k_out) store8<A>(a.k_out, at, k);
  if (a.v_out) store8<A>(a.v_out, at, v);
}

constexpr int kCopyUnroll = 4, kFewPairs = 16;
struct FewPairs {
  int32_t src[kFewPairs], dst[kFewPairs];
};

// A page of a layer is contiguous, nkv * 544 16-byte words: work-groups (x) by
// layer and pair (y), every thread with its words in flight together.  256 pages
// of 28 layers (1 GB read and written): 193-202 us, 5.0 TB/s, as the runtime's own
// device copy; past the caches (nontemporal) 192 us, but eight pages, which fit
// them, 10.1 in place of 5.4 us.  One index range over all words with a division
// for each took 7.0 us there.
template <class PAIRS>
__global__ void __launch_bounds__(256) pkv_copy_kernel(PAIRS p, int layers, int words, const u32x4* src,
                                                       int src_pages, u32x4* dst, int dst_pages) {
  const int pair = blockIdx.y / layers, layer = blockIdx.y - pair * layers;
  const int at = blockIdx.x * (256 * kCopyUnroll) + threadIdx.x;
  const u32x4* from = src + ((size_t)layer * src_pages + p.src[pair]) * words;
  u32x4* to = dst + ((size_t)layer * dst_pages + p.dst[pair]) * words;
  if ((int)(blockIdx.x + 1) * (256 * kCopyUnroll) <= words) {
    u32x4 w[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i) w[i] = from[at + i * 256];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i) to[at + i * 256] = w[i];
  } else {
    for (int i = at; i < words; i += 256) to[i] = from[i];
  }
}

__global__ void pkv_clear_plan_kernel(int32_t* plan) {
  if (threadIdx.x < PH_WORDS) plan[threadIdx.x] = 0;
}

}  // namespace

#define BY_ACT(KERNEL, THREADS)                                                                    \
  do {                                                                                             \
    const dim3 grid(a.rows), block((THREADS + 63) / 64 * 64);                                      \
    if (act == ACT_F32) hipLaunchKernelGGL(KERNEL<ACT_F32>, grid, block, 0, s, a);                 \
    else if (act == ACT_F16) hipLaunchKernelGGL(KERNEL<ACT_F16>, grid, block, 0, s, a);            \
    else hipLaunchKernelGGL(KERNEL<ACT_BF16>, grid, block, 0, s, a);                               \
    return hipGetLastError();                                                                      \
  } while (0)

hipError_t launch_pkv_rope(int act, const RopeFreqs& f, int positions, void* cos, void* sin, hipStream_t s) {
  const dim3 grid((unsigned)(((size_t)positions * (HD / 2) + 255) / 256)), block(256);
  if (act == ACT_F32) hipLaunchKernelGGL(pkv_rope_kernel<ACT_F32>, grid, block, 0, s, f, positions, cos, sin);
  else if (act == ACT_F16) hipLaunchKernelGGL(pkv_rope_kernel<ACT_F16>, grid, block, 0, s, f, positions, cos, sin);
  else hipLaunchKernelGGL(pkv_rope_kernel<ACT_BF16>, grid, block, 0, s, f, positions, cos, sin);
  return hipGetLastError();
}

hipError_t launch_pkv_append(int act, const PkvRowArgs& a, hipStream_t s) {
  BY_ACT(pkv_append_kernel, 16 * (a.nh + a.nkv));
}
hipError_t launch_pkv_write(int act, const PkvRowArgs& a, hipStream_t s) {
  BY_ACT(pkv_write_kernel, 16 * a.nkv);
}
hipError_t launch_pkv_read(int act, const PkvRowArgs& a, hipStream_t s) {
  BY_ACT(pkv_read_kernel, 16 * a.nkv);
}

hipError_t launch_pkv_copy(const PkvPairs& p, int n, int layers, int nkv, const void* src_pool,
                           int src_pages, void* dst_pool, int dst_pages, hipStream_t s) {
  const int words = nkv * (kPkvHeadBytes / 16), per = 256 * kCopyUnroll;
  if (n < 1 || n > kPkvPairs || (int64_t)n * layers > 65535) return hipErrorInvalidValue;
  const dim3 grid((words + per - 1) / per, n * layers), block(256);
  if (n <= kFewPairs) {
    // few pairs: 128 bytes of kernel arguments in place of 3.6 KB, which a call
    // with its wait shows: 22 against 40 us
    FewPairs f;
    for (int i = 0; i < n; ++i) {
      f.src[i] = p.src[i];
      f.dst[i] = p.dst[i];
    }
    hipLaunchKernelGGL(pkv_copy_kernel<FewPairs>, grid, block, 0, s, f, layers, words,
                       (const u32x4*)src_pool, src_pages, (u32x4*)dst_pool, dst_pages);
  } else {
    hipLaunchKernelGGL(pkv_copy_kernel<PkvPairs>, grid, block, 0, s, p, layers, words,
                       (const u32x4*)src_pool, src_pages, (u32x4*)dst_pool, dst_pages);
  }
  return hipGetLastError();
}

hipError_t launch_pkv_clear_plan(int32_t* plan, hipStream_t s) {
  hipLaunchKernelGGL(pkv_clear_plan_kernel, dim3(1), dim3(64), 0, s, plan);
  return hipGetLastError();
}
