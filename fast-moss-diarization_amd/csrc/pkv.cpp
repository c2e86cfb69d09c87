// The paged 4-bit KV cache: the pool, its plans and the entry points
// (include/fmd_dec.h, fmd_pkv_*); who holds which page is in pkv_pages.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <string>
#include <utility>
#include <vector>

#include "fmd_dec.h"
#include "fmd_internal.h"
#include "fmd_kernels.h"

#define HIPCHK(expr)                                                                   \
  do {                                                                                 \
    hipError_t e_ = (expr);                                                            \
    if (e_ != hipSuccess)                                                              \
      return fmd_fail(FMD_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(e_)); \
  } while (0)
#define CHK(expr)        \
  do {                   \
    int rc_ = (expr);    \
    if (rc_) return rc_; \
  } while (0)

static_assert(FMD_PKV_PAGE == kPkvPage, "page size");
static_assert(PkvPages::kArg == FMD_ERR_ARG && PkvPages::kState == FMD_ERR_STATE &&
                  PkvPages::kOverflow == FMD_ERR_OVERFLOW, "status codes");

struct fmd_pkv {
  fmd_dec* dec = nullptr;
  PkvPages tab;
  DevBuf pool;
  // the current plan
  bool planned = false;
  int rows = 0, ndec = 0, nwork = 0, nsplit = 0;
  DevBuf plan;
  PkvBounds most{};
  int32_t* stage[2] = {nullptr, nullptr};   // pinned; a slot is rewritten once its upload has passed
  hipEvent_t staged[2] = {nullptr, nullptr};
  int slot = 0;
  DevBuf tickets, dec_ml, dec_o, pre_ml, pre_o;      // partial results of rows in several items
};

namespace {

// No C++ exception (host memory running out) leaves a C entry point.
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return fmd_fail(FMD_ERR_OOM, std::string("host: ") + e.what());
  }
}

int check_cache(const fmd_pkv* c) {
  return c ? 0 : fmd_fail(FMD_ERR_ARG, "null handle");
}
// A call on the tables, with its message.
int told(const fmd_pkv* c, int rc) { return rc ? fmd_fail(rc, c->tab.error) : 0; }

int check_idle(const fmd_dec* d) {
  HIPCHK(hipSetDevice(d->device));
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(d->stream, &cap));
  if (cap != hipStreamCaptureStatusNone)
    return fmd_fail(FMD_ERR_STATE, "the cache's pages cannot change under graph capture");
  return 0;
}

// Pages change hands: what was planned over them, captured graphs included,
// finds no rows any more.
int drop_plan(fmd_pkv* c) {
  if (!c->planned) return 0;
  c->planned = false;
  HIPCHK(launch_pkv_clear_plan(c->plan.as<int32_t>(), c->dec->stream));
  return 0;
}

// Copies pages of every layer into the pool from the one at `from`.
int copy_pairs(fmd_pkv* c, const PkvPages::Copies& l, const void* from, int from_pages, void* to,
               int to_pages) {
  fmd_dec* d = c->dec;
  const size_t most = (size_t)std::min(kPkvPairs, 65535 / d->L);   // pairs x layers: the grid's second axis
  if (most == 0) return fmd_fail(FMD_ERR_ARG, "too many layers to copy pages of");
  PkvPairs p;
  for (size_t i = 0; i < l.src.size(); i += most) {
    const size_t n = std::min(most, l.src.size() - i);
    std::copy_n(l.src.begin() + i, n, p.src);
    std::copy_n(l.dst.begin() + i, n, p.dst);
    HIPCHK(launch_pkv_copy(p, (int)n, d->L, d->nkv, from, from_pages, to, to_pages, d->stream));
  }
  return 0;
}

// Synchronous on the handle's own stream outside capture, asynchronous on a
// caller's.
int sync_own(fmd_dec* d) {
  if (d->stream != d->own_stream) return 0;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(d->stream, &cap));
  if (cap == hipStreamCaptureStatusNone) HIPCHK(hipStreamSynchronize(d->stream));
  return 0;
}

int make_tables(fmd_dec* d) {
  if (d->pkv_cos.p && d->pkv_sin.p) return 0;
  const size_t bytes = (size_t)d->max_len * (d->hd / 2) * d->esz;
  CHK(d->pkv_cos.ensure(bytes));
  RopeFreqs f;
  for (int i = 0; i < 64; ++i)   // as fmd_dec_create
    f.inv[i] = (float)(1.0 / std::pow(d->cfg.rope_theta, 2.0 * (double)i / (double)d->hd));
  int rc = d->pkv_sin.ensure(bytes);
  if (!rc && launch_pkv_rope(d->act, f, d->max_len, d->pkv_cos.p, d->pkv_sin.p, d->stream) != hipSuccess) {
    d->pkv_sin.release();
    rc = fmd_fail(FMD_ERR_HIP, "rotation tables failed");
  }
  return rc;
}

int check_op(fmd_dec* d, const fmd_pkv* c, int layer) {
  if (!d || !c) return fmd_fail(FMD_ERR_ARG, "null handle");
  if (c->dec != d) return fmd_fail(FMD_ERR_STATE, "cache belongs to another decoder");
  if (layer < 0 || layer >= d->L) return fmd_fail(FMD_ERR_ARG, "bad layer");
  if (!c->planned) return fmd_fail(FMD_ERR_STATE, "no plan: call fmd_pkv_plan first");
  HIPCHK(hipSetDevice(d->device));
  return 0;
}
int check_aligned(const void* p) {
  return (uintptr_t)p % 16 ? fmd_fail(FMD_ERR_ARG, "device buffers must be 16-byte aligned") : 0;
}

PkvRowArgs row_args(const fmd_pkv* c, int layer) {
  const fmd_dec* d = c->dec;
  PkvRowArgs a{};
  a.plan = c->plan.as<int32_t>();
  a.far = a.plan + c->most.rows_at;
  a.layer = layer;
  a.nh = d->nh;
  a.nkv = d->nkv;
  a.rows = c->rows;
  a.eps = d->eps;
  return a;
}

}  // namespace

// The device part of the two calls of a layer, also used by fmd_dec_step.
int pkv_append(fmd_pkv* c, int layer, const void* qkv, void* q) {
  fmd_dec* d = c->dec;
  if (c->rows == 0) return 0;
  PkvRowArgs a = row_args(c, layer);
  a.x = qkv;
  a.qn_w = d->layers[layer].q_norm;
  a.kn_w = d->layers[layer].k_norm;
  a.cos = d->pkv_cos.p;
  a.sin = d->pkv_sin.p;
  a.q_out = q;
  HIPCHK(launch_pkv_append(d->act, a, d->stream));
  return 0;
}

int pkv_attention(fmd_pkv* c, int layer, const void* q, void* ctx) {
  fmd_dec* d = c->dec;
  if (c->rows == 0) return 0;
  PkvAttnArgs a{};
  a.plan = c->plan.as<int32_t>();
  a.layer = layer;
  a.nkv = d->nkv;
  a.rep = d->rep;
  a.rows = c->rows;
  a.q = q;
  a.out = ctx;
  a.window = c->tab.window;
  a.sinks = c->tab.sinks;
  a.scale = d->scale;
  a.ndec = c->ndec;
  a.nwork = c->nwork;
  a.nsplit = c->nsplit;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(d->stream, &cap));
  a.captured = cap != hipStreamCaptureStatusNone;
  a.tickets = c->tickets.as<uint32_t>();
  a.dec_ml = c->dec_ml.as<float>();
  a.dec_o = c->dec_o.as<float>();
  a.pre_ml = c->pre_ml.as<float>();
  a.pre_o = c->pre_o.as<float>();
  HIPCHK(launch_pkv_attn(d->act, a, d->stream));
  return 0;
}

fmd_dec* pkv_dec(const fmd_pkv* c) { return c->dec; }

extern "C" size_t fmd_pkv_bytes(const fmd_dec* d, int pages) {
  if (!d || pages < 0) return 0;
  return (size_t)d->L * pages * d->nkv * kPkvHeadBytes;
}

extern "C" int fmd_pkv_destroy(fmd_pkv* c) {
  if (!c) return 0;
  hipSetDevice(c->dec->device);
  hipStreamSynchronize(c->dec->stream);
  for (DevBuf* b : {&c->pool, &c->plan, &c->tickets, &c->dec_ml, &c->dec_o, &c->pre_ml, &c->pre_o}) b->release();
  for (int i = 0; i < 2; ++i) {
    if (c->staged[i]) hipEventDestroy(c->staged[i]);
    if (c->stage[i]) hipHostFree(c->stage[i]);
  }
  delete c;
  return 0;
}

extern "C" int fmd_pkv_create(fmd_dec* d, int pages, int max_seqs, int max_rows, int window,
                              int sinks, fmd_pkv** out) {
  if (!d || !out) return fmd_fail(FMD_ERR_ARG, "null argument");
  *out = nullptr;
  if (pages <= 0 || max_seqs <= 0 || max_rows <= 0)
    return fmd_fail(FMD_ERR_ARG, "pages, max_seqs and max_rows must be > 0");
  if (max_seqs > 65536 || max_rows > (1 << 20))
    return fmd_fail(FMD_ERR_ARG, "max_seqs above 65536 or max_rows above 1048576");
  if (window < 0 || sinks < 0) return fmd_fail(FMD_ERR_ARG, "negative window or sinks");
  if (!window && sinks) return fmd_fail(FMD_ERR_ARG, "sinks need a window");
  CHK(check_idle(d));
  fmd_pkv* c = nullptr;
  int rc = guarded([&]() {
    c = new fmd_pkv();
    return 0;
  });
  if (rc) return rc;
  c->dec = d;
  // Everything a plan or a kernel needs is here from the start and never moves
  // (captured graphs hold the addresses): the words of the largest plan, and
  // the partial results of the rows that are cut into items.
  const int tile = pkv_tile_positions(d->act, d->rep);
  c->most = pkv_bounds(d->nkv, max_seqs, max_rows, d->max_len, tile);
  const size_t dec_units = (size_t)c->most.dec_items * d->nkv * d->rep;
  const size_t pre_units = max_rows > 1 ? (size_t)c->most.pre_slots * d->nkv * tile * d->rep : 0;
  rc = make_tables(d);
  if (!rc) rc = c->pool.ensure(fmd_pkv_bytes(d, pages));
  if (!rc) rc = c->plan.ensure(c->most.words * 4);
  if (!rc) rc = c->tickets.ensure((size_t)c->most.dec_items * d->nkv * 4);
  if (!rc) rc = c->dec_ml.ensure(dec_units * 8);
  if (!rc) rc = c->dec_o.ensure(dec_units * d->hd * 4);
  if (!rc) rc = c->pre_ml.ensure(pre_units * 8);
  if (!rc) rc = c->pre_o.ensure(pre_units * d->hd * 4);
  if (!rc)
    rc = guarded([&]() {
      c->tab.init(pages, max_seqs, max_rows, d->max_len, window, sinks);
      return 0;
    });
  for (int i = 0; i < 2 && !rc; ++i) {
    if (hipHostMalloc((void**)&c->stage[i], c->most.words * 4, hipHostMallocDefault) != hipSuccess) {
      (void)hipGetLastError();
      rc = fmd_fail(FMD_ERR_OOM, "pinned allocation failed");
    } else if (hipEventCreateWithFlags(&c->staged[i], hipEventDisableTiming) != hipSuccess) {
      rc = fmd_fail(FMD_ERR_HIP, "event creation failed");
    }
  }
  if (!rc && (launch_pkv_clear_plan(c->plan.as<int32_t>(), d->stream) != hipSuccess ||
              launch_fill_i32(c->tickets.as<int32_t>(), (int64_t)c->most.dec_items * d->nkv, 0, d->stream) !=
                  hipSuccess))
    rc = fmd_fail(FMD_ERR_HIP, "plan clear failed");
  if (!rc && hipStreamSynchronize(d->stream) != hipSuccess) rc = fmd_fail(FMD_ERR_HIP, "sync failed");
  if (rc) {
    const std::string keep = fmd_last_error();
    fmd_pkv_destroy(c);
    return fmd_fail(rc, keep);
  }
  *out = c;
  return 0;
}

extern "C" int fmd_pkv_open(fmd_pkv* c, int32_t* seq) {
  CHK(check_cache(c));
  if (!seq) return fmd_fail(FMD_ERR_ARG, "null argument");
  return told(c, c->tab.open(seq));
}

extern "C" int fmd_pkv_fork(fmd_pkv* c, int seq, int32_t* out) {
  CHK(check_cache(c));
  if (!out) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(told(c, c->tab.check(seq)));
  CHK(check_idle(c->dec));
  CHK(guarded([&]() { return told(c, c->tab.fork(seq, out)); }));
  return drop_plan(c);   // the planned rows of `seq` would land in pages that are now shared
}

extern "C" int fmd_pkv_copy(fmd_pkv* c, int seq, int32_t* out) {
  CHK(check_cache(c));
  if (!out) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(told(c, c->tab.check(seq)));
  CHK(check_idle(c->dec));
  return guarded([&]() {
    PkvPages::Copies l;
    int32_t made = -1;
    CHK(told(c, c->tab.copy(seq, &made, &l)));
    const int rc = copy_pairs(c, l, c->pool.p, c->tab.pages, c->pool.p, c->tab.pages);
    if (rc) {
      c->tab.free(made);
      return rc;
    }
    *out = made;
    return sync_own(c->dec);
  });
}

extern "C" int fmd_pkv_free(fmd_pkv* c, int seq) {
  CHK(check_cache(c));
  CHK(told(c, c->tab.check(seq)));
  CHK(check_idle(c->dec));
  CHK(guarded([&]() { return told(c, c->tab.free(seq)); }));
  return drop_plan(c);
}

extern "C" int fmd_pkv_truncate(fmd_pkv* c, int seq, int len) {
  CHK(check_cache(c));
  CHK(told(c, c->tab.check(seq)));
  CHK(check_idle(c->dec));
  const int before = c->tab.seqs[seq].len;
  return guarded([&]() {
    CHK(told(c, c->tab.truncate(seq, len)));
    return len == before ? 0 : drop_plan(c);
  });
}

extern "C" int fmd_pkv_resize(fmd_pkv* c, int pages) {
  CHK(check_cache(c));
  CHK(check_idle(c->dec));
  return guarded([&]() {
    const bool in_place = pages == c->tab.pages;
    std::vector<int32_t> to;
    PkvPages::Copies l;
    CHK(told(c, c->tab.compaction(pages, !in_place, &to, &l)));
    if (in_place && l.src.empty()) return 0;
    CHK(drop_plan(c));
    DevBuf fresh;
    if (!in_place) CHK(fresh.ensure(fmd_pkv_bytes(c->dec, pages)));
    int rc = copy_pairs(c, l, c->pool.p, c->tab.pages, in_place ? c->pool.p : fresh.p, pages);
    if (!rc && hipStreamSynchronize(c->dec->stream) != hipSuccess)
      rc = fmd_fail(FMD_ERR_HIP, "page copy failed");
    if (!rc) {
      c->tab.compacted(pages, to);
      if (!in_place) std::swap(fresh, c->pool);
    }
    fresh.release();
    return rc;
  });
}

extern "C" int fmd_pkv_len(const fmd_pkv* c, int seq) {
  if (check_cache(c)) return -1;
  if (seq < 0 || seq >= (int)c->tab.seqs.size() || !c->tab.seqs[seq].open) {
    fmd_fail(FMD_ERR_ARG, "no such sequence");
    return -1;
  }
  return c->tab.seqs[seq].len;
}
extern "C" int fmd_pkv_free_pages(const fmd_pkv* c) { return c ? c->tab.free_pages() : -1; }

extern "C" int fmd_pkv_pages(const fmd_pkv* c, int seq, int32_t* out, int room, int32_t* n) {
  if (fmd_pkv_len(c, seq) < 0) return FMD_ERR_ARG;
  if (!n || (room > 0 && !out)) return fmd_fail(FMD_ERR_ARG, "null argument");
  const std::vector<int32_t>& p = c->tab.seqs[seq].pages;
  *n = (int32_t)p.size();
  for (int i = 0; i < room && i < (int)p.size(); ++i) out[i] = p[i];
  return 0;
}

extern "C" int fmd_pkv_pool(const fmd_pkv* c, void** data, size_t* bytes) {
  CHK(check_cache(c));
  if (!data || !bytes) return fmd_fail(FMD_ERR_ARG, "null argument");
  *data = c->pool.p;
  *bytes = fmd_pkv_bytes(c->dec, c->tab.pages);
  return 0;
}

extern "C" int fmd_pkv_plan(fmd_pkv* c, int n, const int32_t* seqs, const int32_t* counts) {
  CHK(check_cache(c));
  CHK(check_idle(c->dec));
  return guarded([&]() {
    fmd_dec* d = c->dec;
    PkvPages::Copies l;
    CHK(told(c, c->tab.extend(n, seqs, counts, &l)));
    CHK(drop_plan(c));
    CHK(copy_pairs(c, l, c->pool.p, c->tab.pages, c->pool.p, c->tab.pages));
    std::vector<int32_t> far;
    std::vector<int32_t> w =
        pkv_build_plan(c->tab, d->nkv, pkv_tile_positions(d->act, d->rep), n, seqs, counts, &far);
    if (w.size() > c->most.rows_at || w[PH_NDEC] > c->most.dec_items)
      return fmd_fail(FMD_ERR_STATE, "plan larger than its buffer");
    const uint64_t pool = (uint64_t)(uintptr_t)c->pool.p;
    w[PH_POOL] = (int32_t)(uint32_t)pool;
    w[PH_POOL + 1] = (int32_t)(uint32_t)(pool >> 32);
    HIPCHK(hipEventSynchronize(c->staged[c->slot]));
    std::memcpy(c->stage[c->slot], w.data(), w.size() * 4);
    HIPCHK(hipMemcpyAsync(c->plan.p, c->stage[c->slot], w.size() * 4, hipMemcpyHostToDevice, d->stream));
    if (!far.empty()) {
      const size_t at = c->most.rows_at;
      std::memcpy(c->stage[c->slot] + at, far.data(), far.size() * 4);
      HIPCHK(hipMemcpyAsync(c->plan.as<int32_t>() + at, c->stage[c->slot] + at, far.size() * 4,
                            hipMemcpyHostToDevice, d->stream));
    }
    HIPCHK(hipEventRecord(c->staged[c->slot], d->stream));
    c->slot ^= 1;
    c->rows = w[PH_ROWS];
    c->ndec = w[PH_NDEC];
    c->nwork = w[PH_NWORK];
    c->nsplit = w[PH_NSPLIT];
    c->planned = true;
    return 0;
  });
}

extern "C" int fmd_op_pkv_append(fmd_dec* d, fmd_pkv* c, int layer, const void* qkv, void* q) {
  CHK(check_op(d, c, layer));
  if (!qkv || !q) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(check_aligned(qkv));
  CHK(check_aligned(q));
  constexpr uint32_t kNorms = (1u << 9) | (1u << 10);   // q_norm, k_norm (resolve in fmd_dec.cpp)
  if ((d->layers[layer].set & kNorms) != kNorms)
    return fmd_fail(FMD_ERR_STATE, "the layer's q_norm and k_norm are not set");
  CHK(pkv_append(c, layer, qkv, q));
  return sync_own(d);
}

extern "C" int fmd_op_pkv_write(fmd_dec* d, fmd_pkv* c, int layer, const void* k, const void* v) {
  CHK(check_op(d, c, layer));
  if (!k || !v) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(check_aligned(k));
  CHK(check_aligned(v));
  if (c->rows == 0) return 0;
  PkvRowArgs a = row_args(c, layer);
  a.x = k;
  a.v = v;
  HIPCHK(launch_pkv_write(d->act, a, d->stream));
  return sync_own(d);
}

extern "C" int fmd_op_pkv_read(fmd_dec* d, fmd_pkv* c, int layer, void* k, void* v) {
  CHK(check_op(d, c, layer));
  if (!k && !v) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(check_aligned(k));
  CHK(check_aligned(v));
  if (c->rows == 0) return 0;
  PkvRowArgs a = row_args(c, layer);
  a.k_out = k;
  a.v_out = v;
  HIPCHK(launch_pkv_read(d->act, a, d->stream));
  return sync_own(d);
}

extern "C" int fmd_op_pkv_attention(fmd_dec* d, fmd_pkv* c, int layer, const void* q, void* ctx) {
  CHK(check_op(d, c, layer));
  if (!q || !ctx) return fmd_fail(FMD_ERR_ARG, "null argument");
  CHK(check_aligned(q));
  CHK(check_aligned(ctx));
  CHK(pkv_attention(c, layer, q, ctx));
  return sync_own(d);
}

extern "C" int fmd_op_pkv_copy_pages(fmd_pkv* c, int n, const int32_t* src, const int32_t* dst) {
  CHK(check_cache(c));
  if (n < 0 || (n > 0 && (!src || !dst))) return fmd_fail(FMD_ERR_ARG, "bad argument");
  HIPCHK(hipSetDevice(c->dec->device));
  return guarded([&]() {
    const int pages = c->tab.pages;
    std::vector<char> role(pages, 0);   // 1 source, 2 destination
    for (int i = 0; i < n; ++i) {
      if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
        return fmd_fail(FMD_ERR_ARG, "page outside the pool");
      role[src[i]] = 1;
    }
    for (int i = 0; i < n; ++i) {
      if (role[dst[i]]) return fmd_fail(FMD_ERR_ARG, "a destination page is named twice or is a source");
      role[dst[i]] = 2;
    }
    if (n == 0) return 0;
    PkvPages::Copies l;
    l.src.assign(src, src + n);
    l.dst.assign(dst, dst + n);
    CHK(copy_pairs(c, l, c->pool.p, pages, c->pool.p, pages));
    return sync_own(c->dec);
  });
}
