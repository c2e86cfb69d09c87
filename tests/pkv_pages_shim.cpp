// C entry points over csrc/pkv_pages.h, for tests/test_pkv_pages.py.
#include "pkv_pages.h"

static PkvPages::Copies g_copies;
static std::vector<int32_t> g_plan, g_far, g_to;

extern "C" {
void* pages_new(int pages, int seqs, int rows, int max_len, int window, int sinks) {
  PkvPages* p = new PkvPages();
  p->init(pages, seqs, rows, max_len, window, sinks);
  return p;
}
void pages_delete(void* p) { delete (PkvPages*)p; }
const char* pages_error(void* p) { return ((PkvPages*)p)->error.c_str(); }
int pages_open(void* p, int32_t* out) { return ((PkvPages*)p)->open(out); }
int pages_fork(void* p, int s, int32_t* out) { return ((PkvPages*)p)->fork(s, out); }
int pages_copy(void* p, int s, int32_t* out) {
  g_copies = {};
  return ((PkvPages*)p)->copy(s, out, &g_copies);
}
int pages_free(void* p, int s) { return ((PkvPages*)p)->free(s); }
int pages_truncate(void* p, int s, int len) { return ((PkvPages*)p)->truncate(s, len); }
int pages_extend(void* p, int n, const int32_t* seqs, const int32_t* counts) {
  g_copies = {};
  return ((PkvPages*)p)->extend(n, seqs, counts, &g_copies);
}
int pages_compact(void* p, int pages, int all) {
  g_copies = {};
  PkvPages* c = (PkvPages*)p;
  if (int rc = c->compaction(pages, all, &g_to, &g_copies)) return rc;
  c->compacted(pages, g_to);
  return 0;
}
int copies_n() { return (int)g_copies.src.size(); }
const int32_t* copies_src() { return g_copies.src.data(); }
const int32_t* copies_dst() { return g_copies.dst.data(); }
int pages_len(void* p, int s) { return ((PkvPages*)p)->seqs[s].len; }
int pages_n(void* p, int s) { return (int)((PkvPages*)p)->seqs[s].pages.size(); }
const int32_t* pages_of(void* p, int s) { return ((PkvPages*)p)->seqs[s].pages.data(); }
const int32_t* pages_refs(void* p) { return ((PkvPages*)p)->refs.data(); }
int pages_free_n(void* p) { return ((PkvPages*)p)->free_pages(); }
int pages_plan(void* p, int nkv, int tile, int n, const int32_t* seqs, const int32_t* counts) {
  g_plan = pkv_build_plan(*(PkvPages*)p, nkv, tile, n, seqs, counts, &g_far);
  return (int)g_plan.size();
}
const int32_t* plan_words() { return g_plan.data(); }
int plan_far(const int32_t** out) {
  *out = g_far.data();
  return (int)g_far.size();
}
void plan_bounds(int nkv, int seqs, int rows, int max_len, int tile, int64_t* out) {
  const PkvBounds b = pkv_bounds(nkv, seqs, rows, max_len, tile);
  out[0] = b.dec_items;
  out[1] = b.tiles;
  out[2] = b.pre_slots;
  out[3] = (int64_t)b.rows_at;
  out[4] = (int64_t)b.words;
}
}
