// The paged 4-bit KV cache on the host: which sequence holds which pages, and
// the plan (include/fmd_dec.h, fmd_pkv_*) as the kernels read it.  Plain C++,
// without a device.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <queue>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

// A page holds 64 tokens of one layer.  Of each KV head it holds 8704 bytes:
//   K codes   4096  [64 tokens][64 B]: dim d in byte d/2, even dims low
//   V codes   4096  the same
//   K scales   256  block b (dims 32b ..) of token t at 64 b + 4 (4 (t/16) + t%4) + (t%16)/4
//   V scales   256  block b of token t at 64 b + t
// Codes are e2m1 (sign, two exponent bits, one mantissa bit), scales 2^(byte -
// 127) with 255 for "not a number".  The K scales of the four tokens that a
// lane's score tiles need (pkv_attn.hip) are one word, the V scales of the 16
// tokens it weighs are 16 bytes.
constexpr int kPkvPage = 64;
constexpr int kPkvHeadBytes = 8704;
constexpr int kPkvV = 4096, kPkvKs = 8192, kPkvVs = 8448;

// The plan in device memory (32-bit words): the header, then position and page
// of each row of a plan of at most kPkvDirect rows, then the decode items, and
// at header offsets the other sections.  The rows of a larger plan are at
// PkvBounds::rows_at: a second upload, which small plans do without.
constexpr int kPkvDirect = 256;
enum PkvHdr {
  PH_ROWS = 0,     // rows of the plan; 0 when there is no plan
  PH_POOL = 1,     // pool address, low and high word
  PH_PAGES = 3,    // pages of the pool (the layer stride)
  PH_NDEC = 4,     // decode items, behind the rows
  PH_NWORK = 5,    // work-groups per KV head of the many-token rows
  PH_NSPLIT = 6,   // many-token tiles in several items
  PH_WORK = 7,     // offset: first item of each of those work-groups, and the item count
  PH_PITEM = 8,    // offset: PkvPreItem entries
  PH_SPLIT = 9,    // offset: PkvSplit entries
  PH_WORDS = 32,
  PH_ITEMS = PH_WORDS + 2 * kPkvDirect
};
// The visible pages of an item's queries, in order: pages [0, sp) (the sinks),
// then pages wp, wp + 1, ..; v counts through both.
struct PkvDecItem {
  int32_t row, pos, table, sp, wp, v0, v1;
  int32_t slot, first, parts;                      // its partial slot, of first .. first + parts - 1 of its row
  int32_t id[4];                                   // the first pages of its four waves
  int32_t pad[2];
};
struct PkvPreItem {
  int32_t row, pos, n, table, sp, wp, v0, v1, slot, pad[3];
};
struct PkvSplit {
  int32_t row, n, first, parts;
};

inline int pkv_ceil(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Sequences and pages.  Calls return 0 or an FMD_ERR_* code with `error` set;
// a failed call has changed nothing.
class PkvPages {
 public:
  static constexpr int kArg = -1, kState = -2, kOverflow = -5;   // FMD_ERR_ARG, _STATE, _OVERFLOW
  struct Seq {
    bool open = false;
    int len = 0;
    std::vector<int32_t> pages;   // -1: released (behind the window)
  };
  struct Copies {
    std::vector<int32_t> src, dst;
  };

  std::string error;
  int pages = 0, max_rows = 0, max_len = 0, window = 0, sinks = 0;
  std::vector<int32_t> refs;
  std::vector<Seq> seqs;

  void init(int pages_, int max_seqs, int max_rows_, int max_len_, int window_, int sinks_) {
    pages = pages_;
    max_rows = max_rows_;
    max_len = max_len_;
    window = window_;
    sinks = sinks_;
    seqs.assign(max_seqs, Seq());
    refs.assign(pages, 0);
    free_ids_ = {};
    for (int i = 0; i < pages; ++i) free_ids_.push(i);
  }
  int free_pages() const { return (int)free_ids_.size(); }
  int live_pages() const { return pages - free_pages(); }

  int check(int seq) {
    if (seq < 0 || seq >= (int)seqs.size() || !seqs[seq].open)
      return fail(kArg, "no such sequence: " + std::to_string(seq));
    return 0;
  }
  int open(int32_t* out) {
    int i = 0;
    while (i < (int)seqs.size() && seqs[i].open) ++i;
    if (i == (int)seqs.size()) return fail(kOverflow, "every sequence of the cache is open");
    seqs[i] = Seq();
    seqs[i].open = true;
    *out = i;
    return 0;
  }
  int fork(int seq, int32_t* out) {
    if (int rc = check(seq)) return rc;
    if (int rc = open(out)) return rc;
    Seq s = seqs[seq];
    for (int32_t id : s.pages)
      if (id >= 0) ++refs[id];
    seqs[*out] = std::move(s);
    return 0;
  }
  int copy(int seq, int32_t* out, Copies* c) {
    if (int rc = check(seq)) return rc;
    Seq s = seqs[seq];
    int n = 0;
    for (int32_t id : s.pages) n += id >= 0;
    if (n > free_pages()) return no_pages(n);
    if (int rc = open(out)) return rc;
    for (int32_t& id : s.pages)
      if (id >= 0) {
        c->src.push_back(id);
        c->dst.push_back(id = take());
      }
    seqs[*out] = std::move(s);
    return 0;
  }
  int free(int seq) {
    if (int rc = check(seq)) return rc;
    for (int32_t id : seqs[seq].pages) drop(id);
    seqs[seq] = Seq();
    return 0;
  }
  int truncate(int seq, int len) {
    if (int rc = check(seq)) return rc;
    Seq& s = seqs[seq];
    if (len < 0 || len > s.len) return fail(kArg, "length outside the sequence");
    const int keep = pkv_ceil(len, kPkvPage);
    for (int p = window_lo(len) / kPkvPage; p < keep; ++p)
      if (s.pages[p] < 0)
        return fail(kState, "the window at position " + std::to_string(len) +
                                " holds tokens whose pages were released");
    for (size_t p = keep; p < s.pages.size(); ++p) drop(s.pages[p]);
    s.pages.resize(keep);
    s.len = len;
    return 0;
  }

  // Where each live page goes when they are moved to the front: those already
  // there stay, the others take the free places (no page is both read and
  // written).  With all, pages that stay are listed too (a move to a new pool).
  int compaction(int new_pages, bool all, std::vector<int32_t>* to, Copies* c) {
    const int live = live_pages();
    if (new_pages <= 0 || new_pages < live)
      return fail(kArg, std::to_string(live) + " pages are in use; a pool of " +
                            std::to_string(new_pages) + " cannot hold them");
    to->assign(pages, -1);
    for (int i = 0, at = 0; i < pages; ++i) {
      if (refs[i] == 0) continue;
      if (i < live) {
        (*to)[i] = i;
      } else {
        while (refs[at] > 0) ++at;
        (*to)[i] = at++;
      }
      if (all || (*to)[i] != i) {
        c->src.push_back(i);
        c->dst.push_back((*to)[i]);
      }
    }
    return 0;
  }
  void compacted(int new_pages, const std::vector<int32_t>& to) {
    const int live = live_pages();
    std::vector<int32_t> r(new_pages, 0);
    for (size_t i = 0; i < to.size(); ++i)
      if (to[i] >= 0) r[to[i]] = refs[i];
    refs = std::move(r);
    pages = new_pages;
    free_ids_ = {};
    for (int i = live; i < pages; ++i) free_ids_.push(i);
    for (Seq& s : seqs)
      for (int32_t& id : s.pages)
        if (id >= 0) id = to[id];
  }

  // counts[i] new tokens for seqs[i]: pages behind the windows are given back,
  // shared pages that will be written to are replaced (in *c), new ones taken.
  int extend(int n, const int32_t* which, const int32_t* counts, Copies* c) {
    if (n < 0 || n > (int)seqs.size()) return fail(kArg, "more sequences than the cache holds");
    if (n > 0 && (!which || !counts)) return fail(kArg, "null argument");
    std::vector<char> seen(seqs.size(), 0);
    int64_t rows = 0;
    for (int i = 0; i < n; ++i) {
      if (int rc = check(which[i])) return rc;
      if (seen[which[i]]++) return fail(kArg, "sequence " + std::to_string(which[i]) + " is named twice");
      if (counts[i] < 0) return fail(kArg, "negative token count");
      if ((int64_t)seqs[which[i]].len + counts[i] > max_len)
        return fail(kArg, "position beyond the RoPE table");
      rows += counts[i];
    }
    if (rows > max_rows)
      return fail(kArg, std::to_string(rows) + " new tokens; the cache was made for " +
                            std::to_string(max_rows) + " at a time");
    // before anything changes: do the pages suffice?
    std::unordered_map<int32_t, int> given;   // references that go, by page
    int64_t need = 0, freed = 0;
    for (int i = 0; i < n; ++i) {
      const Seq& s = seqs[which[i]];
      for (int p = 0; counts[i] && window && p < (int)s.pages.size(); ++p)
        if (s.pages[p] >= 0 && behind(p, s.len) && ++given[s.pages[p]] == refs[s.pages[p]]) ++freed;
    }
    for (int i = 0; i < n; ++i) {
      const Seq& s = seqs[which[i]];
      if (!counts[i]) continue;
      need += pkv_ceil(s.len + counts[i], kPkvPage) - (int)s.pages.size();
      if (s.len % kPkvPage) {
        // the page of the last token, never behind the window of the next one;
        // the last holder writes in place
        const int32_t id = s.pages.back();
        if (refs[id] - given[id] > 1) {
          ++given[id];
          ++need;
        }
      }
    }
    if (need > (int64_t)free_pages() + freed) return no_pages((int)std::min<int64_t>(need, INT32_MAX));
    for (int i = 0; i < n; ++i) {
      Seq& s = seqs[which[i]];
      for (int p = 0; counts[i] && window && p < (int)s.pages.size(); ++p)
        if (s.pages[p] >= 0 && behind(p, s.len)) {
          drop(s.pages[p]);
          s.pages[p] = -1;
        }
    }
    for (int i = 0; i < n; ++i) {
      Seq& s = seqs[which[i]];
      if (!counts[i]) continue;
      if (s.len % kPkvPage && refs[s.pages.back()] > 1) {
        c->src.push_back(s.pages.back());
        --refs[s.pages.back()];
        s.pages.back() = take();
        c->dst.push_back(s.pages.back());
      }
      s.len += counts[i];
      while ((int64_t)s.pages.size() * kPkvPage < s.len) s.pages.push_back(take());
    }
    return 0;
  }

  // First key of the window of a query at position pos.
  int window_lo(int pos) const { return window ? std::max(0, pos - window + 1) : 0; }
  // No query at position len or later sees the page.
  bool behind(int page, int len) const {
    return (int64_t)(page + 1) * kPkvPage <= window_lo(len) && (int64_t)page * kPkvPage >= sinks;
  }
  // The pages that queries at positions pos .. last see: [0, sp) and the n - sp from wp on.
  struct Visible {
    int sp, wp, n;
  };
  Visible visible(int pos, int last) const {
    Visible v;
    v.wp = window_lo(pos) / kPkvPage;
    v.sp = std::min(v.wp, pkv_ceil(std::min(sinks, pos + 1), kPkvPage));
    v.n = v.sp + last / kPkvPage + 1 - v.wp;
    return v;
  }

 private:
  std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free_ids_;   // lowest first

  int fail(int code, const std::string& msg) {
    error = msg;
    return code;
  }
  int no_pages(int need) {
    return fail(kOverflow, "paged kv cache overflow: " + std::to_string(need) + " pages needed, " +
                               std::to_string(free_pages()) + " of " + std::to_string(pages) + " free");
  }
  int32_t take() {
    const int32_t id = free_ids_.top();
    free_ids_.pop();
    refs[id] = 1;
    return id;
  }
  void drop(int32_t id) {
    if (id >= 0 && --refs[id] == 0) free_ids_.push(id);
  }
};

// ---- the plan ----

// Work-groups that the attention is cut for, over all KV heads (two on each CU),
// and the pages of a decode item and a many-token work-group at least: two of each
// decode wave's cost less than handing one over (one row of 450 keys at 4 | 8
// pages: 6.7 | 6.5 us), and below eight a many-token run is shorter than its
// partial result is worth.
constexpr int kPkvDecGroups = 512, kPkvPreGroups = 512;
constexpr int kPkvDecMinPages = 8, kPkvPreMinPages = 8;

// What a plan takes at most.  Decode: an item's pages are at least all rows'
// pages over kPkvDecGroups / nkv, so there are at most that many items and one
// more per row.  Many tokens: the tiles' pages, one tile after another, are cut
// into equal runs for the work-groups; a cut adds an item and makes two partial.
struct PkvBounds {
  int dec_items, tiles, pre_slots;
  size_t rows_at;   // the rows of plans of more than kPkvDirect
  size_t words;
};
inline PkvBounds pkv_bounds(int nkv, int max_seqs, int max_rows, int max_len, int tile) {
  PkvBounds b;
  b.dec_items = kPkvDecGroups / nkv + max_seqs + 1;
  b.tiles = max_rows / tile + max_seqs;
  b.pre_slots = 2 * (kPkvPreGroups / nkv + 1);
  b.rows_at = PH_ITEMS + ((size_t)b.dec_items * sizeof(PkvDecItem) +
                          (size_t)(b.tiles + b.pre_slots) * sizeof(PkvPreItem) +
                          (size_t)b.pre_slots * (sizeof(PkvSplit) + 4)) / 4 +
              (size_t)max_seqs * pkv_ceil(max_len, kPkvPage);
  b.words = b.rows_at + (max_rows > kPkvDirect ? 2 * (size_t)max_rows : 0);
  return b;
}

// The plan of the last counts[i] tokens of seqs[i], `tile` positions to a
// many-token tile; the pool's address goes into the header later.  The rows of a
// plan of more than kPkvDirect are left in *far.
inline std::vector<int32_t> pkv_build_plan(const PkvPages& c, int nkv, int tile, int n, const int32_t* seqs,
                                           const int32_t* counts, std::vector<int32_t>* far) {
  struct Row {
    int seq, row, pos, n;
  };
  std::vector<Row> order;
  int64_t dec_pages = 0, pre_pages = 0;
  int rows = 0;
  for (int i = 0; i < n; ++i) {
    const int pos = c.seqs[seqs[i]].len - counts[i];
    order.push_back({seqs[i], rows, pos, counts[i]});
    if (counts[i] == 1) dec_pages += c.visible(pos, pos).n;
    for (int p = 0; counts[i] > 1 && p < counts[i]; p += tile)
      pre_pages += c.visible(pos + p, pos + std::min(p + tile, counts[i]) - 1).n;
    rows += counts[i];
  }
  std::vector<PkvDecItem> di;
  std::vector<PkvPreItem> pi;
  std::vector<PkvSplit> sp;
  std::vector<int32_t> toff(n, 0), table;
  // as many pages to an item as it takes for the items to fit the device's
  // work-group slots in one round, if they can
  int dec_per = std::max(kPkvDecMinPages, pkv_ceil(dec_pages * nkv, kPkvDecGroups));
  auto dec_items = [&]() {
    int64_t k = 0;
    for (const Row& r : order)
      if (r.n == 1) k += pkv_ceil(c.visible(r.pos, r.pos).n, dec_per);
    return k;
  };
  int dec_rows = 0;
  for (const Row& r : order) dec_rows += r.n == 1;
  while ((int64_t)dec_rows * nkv <= kPkvDecGroups && dec_items() * nkv > kPkvDecGroups)
    dec_per += std::max(1, dec_per / 16);
  const int pre_per = std::max(kPkvPreMinPages, pkv_ceil(pre_pages, std::max(1, kPkvPreGroups / nkv)));
  int dec_slots = 0, pre_slots = 0, room = pre_per;   // pages that the work-group at hand still takes
  std::vector<int32_t> work(1, 0);
  for (int i = 0; i < n; ++i) {
    const Row& r = order[i];
    toff[i] = (int)table.size();
    if (r.n) table.insert(table.end(), c.seqs[r.seq].pages.begin(), c.seqs[r.seq].pages.end());
    if (r.n == 1) {
      const PkvPages::Visible v = c.visible(r.pos, r.pos);
      const int per = pkv_ceil(v.n, pkv_ceil(v.n, dec_per)), parts = pkv_ceil(v.n, per);
      for (int k = 0; k < parts; ++k) {
        PkvDecItem x{r.row, r.pos, i, v.sp, v.wp, k * per, std::min((k + 1) * per, v.n), dec_slots + k,
                     dec_slots, parts, {0, 0, 0, 0}, {0, 0}};
        for (int j = 0; j < 4; ++j) {
          const int at = std::min(x.v0 + j, x.v1 - 1);
          x.id[j] = c.seqs[r.seq].pages[at < v.sp ? at : v.wp + at - v.sp];
        }
        di.push_back(x);
      }
      dec_slots += parts;
    } else {
      for (int p = 0; p < r.n; p += tile) {
        const int m = std::min(tile, r.n - p);
        const PkvPages::Visible v = c.visible(r.pos + p, r.pos + p + m - 1);
        const bool whole = v.n <= room;
        int parts = 0;
        for (int v0 = 0; v0 < v.n; ++parts) {
          const int k = std::min(room, v.n - v0);
          pi.push_back({r.row + p, r.pos + p, m, i, v.sp, v.wp, v0, v0 + k, whole ? -1 : pre_slots + parts, {0, 0, 0}});
          v0 += k;
          room -= k;
          if (room == 0) {
            work.push_back((int)pi.size());
            room = pre_per;
          }
        }
        if (!whole) {
          sp.push_back({r.row + p, m, pre_slots, parts});
          pre_slots += parts;
        }
      }
    }
  }
  if (work.back() != (int)pi.size()) work.push_back((int)pi.size());
  std::vector<int32_t> w(PH_ITEMS, 0);
  auto section = [&](size_t words) {
    const int at = (int)w.size();
    w.resize(w.size() + words);
    return at;
  };
  auto put = [&](const void* src, size_t words) {
    const int at = section(words);
    if (words) std::memcpy(w.data() + at, src, words * 4);
    return at;
  };
  // the sections' sizes are known: the tables come last, behind `table_at`
  const size_t di_words = di.size() * sizeof(PkvDecItem) / 4,
               pi_words = pi.size() * sizeof(PkvPreItem) / 4, sp_words = sp.size() * sizeof(PkvSplit) / 4;
  const int table_at = (int)(PH_ITEMS + di_words + pi_words + work.size() + sp_words);
  for (PkvDecItem& x : di) x.table = table_at + toff[x.table];
  for (PkvPreItem& x : pi) x.table = table_at + toff[x.table];
  put(di.data(), di_words);
  w[PH_PITEM] = put(pi.data(), pi_words);
  w[PH_WORK] = put(work.data(), work.size());
  w[PH_SPLIT] = put(sp.data(), sp_words);
  put(table.data(), table.size());
  w[PH_ROWS] = rows;
  w[PH_PAGES] = c.pages;
  w[PH_NDEC] = (int)di.size();
  w[PH_NWORK] = (int)work.size() - 1;
  w[PH_NSPLIT] = (int)sp.size();
  far->assign(rows > kPkvDirect ? 2 * (size_t)rows : 0, 0);
  int32_t* at = rows > kPkvDirect ? far->data() : w.data() + PH_WORDS;
  for (const Row& r : order)
    for (int k = 0; k < r.n; ++k) {
      *at++ = r.pos + k;
      *at++ = c.seqs[r.seq].pages[(r.pos + k) / kPkvPage];
    }
  return w;
}
