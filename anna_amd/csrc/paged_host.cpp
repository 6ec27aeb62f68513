// The paged 4-bit cache's host side: which pages are whose, and the plans of its launches.
//
// The free pages are a stack, so that a sequence that ends gives its pages to the next one; a page
// carries the number of sequences that hold it and is copied when one of several holders writes
// into it.  Every call checks all its arguments before it changes anything.
#include <limits.h>
#include <stddef.h>

#include <algorithm>
#include <memory>
#include <mutex>
#include <new>
#include <vector>

#include "paged.hpp"

using namespace anna;
using namespace anna::paged;

struct anna_mi_paged {
  std::mutex lock;
  anna_mi_paged_desc d;
  std::vector<int32_t> table;   // [max_sequences][max_pages]
  std::vector<int64_t> length;  // -1: not in use
  std::vector<int32_t> refs;    // of every page
  std::vector<int32_t> free_pages, free_seqs;
  std::vector<uint8_t> seen;  // by sequence, zero between calls
  // of an extend whose launch is left to the span's fill: table entries (index, page) and page copies (source, page)
  std::vector<int32_t> entries, pairs;

  int32_t* row(int64_t seq) { return table.data() + seq * d.max_pages; }
  int64_t pages(int64_t seq) const { return (length[seq] + PAGE - 1) / PAGE; }
  int64_t page_size() const { return d.kv_heads * page_bytes(d.head_dim); }
};

namespace {

// Workgroups of a launch that run at once on the 256 compute units: two on each of the split form, one of the tile
// form.  A few more than that would leave most of the chip idle for a whole round: with up to 640 and 512 of them drafted
// tokens take 50 us, not 42, 8 sequences of 1K to 16K 27, not 24, 2048 tokens at the end of 32K 1196, not 1166.
constexpr int64_t SPLIT_ONCE = 512, TILE_ONCE = 256;
// Tiles of 256 rows when they fill the chip; an item of the tile form has TILE_PAGES pages at least, as its partial
// result is written and read again; up to TILE_LEAST query rows of a KV head are the split form's.
constexpr int64_t TILE_FILL = 256, TILE_PAGES = 8, TILE_LEAST = 64;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of a launch, of up to 512 threads: 32 bits count its threads.
constexpr int64_t MOST_GROUPS = UINT_MAX / 512;

int hip_ok(hipError_t e, const char* what) { return e == hipSuccess ? ANNA_MI_OK : fail_hip(e, what); }

// Batches words of the four kinds into as few launches as they need.
struct Updates {
  Update u;
  hipStream_t stream;
  std::vector<int32_t> records, entries, copies, pairs;
  Updates(anna_mi_paged* h, void* s) : stream(as_stream(s)) {
    memset(&u, 0, offsetof(Update, words));
    u.table = h->d.table;
    u.width = h->d.max_pages;
    u.pool = (uint8_t*)h->d.pool;
    u.page = h->page_size();
    u.pool_layer = h->d.num_pages * u.page;
    u.layers = (int32_t)h->d.num_layers;
  }
  void entry(int64_t index, int32_t page) { entries.insert(entries.end(), {(int32_t)index, page}); }
  void copy(int32_t row, int32_t source, int64_t pages) { copies.insert(copies.end(), {row, source, (int32_t)pages}); }
  int launch() {
    constexpr int R = sizeof(Record) / 4;
    size_t r = 0, e = 0, c = 0, p = 0;
    while (r < records.size() || e < entries.size() || c < copies.size() || p < pairs.size()) {
      int n = 0;
      auto take = [&](const std::vector<int32_t>& v, size_t& at, int step, size_t most = UPDATE_WORDS) {
        const int k = (int)std::min({(v.size() - at) / step, (size_t)(UPDATE_WORDS - n) / step, most});
        if (k > 0) memcpy(u.words + n, v.data() + at, 4 * (size_t)k * step);
        n += k * step;
        at += (size_t)k * step;
        return k;
      };
      u.records = take(records, r, R);
      u.entries = take(entries, e, 2);
      u.copies = take(copies, c, 3);
      u.pairs = take(pairs, p, 2, std::max<int64_t>(1, MOST_GROUPS / 2 / (u.layers * ceil_div(u.page, COPY_BYTES))));
      const int rc = launch_update(u, stream);
      if (rc != ANNA_MI_OK) return rc;
    }
    return ANNA_MI_OK;
  }
};

// What an extend left to a span's fill, for any other call that comes first.
int flush(anna_mi_paged* h, void* stream) {
  if (h->entries.empty() && h->pairs.empty()) return ANNA_MI_OK;
  Updates up(h, stream);
  up.entries.swap(h->entries);
  up.pairs.swap(h->pairs);
  return up.launch();
}

// pairs: (source, page), ...
int copy_pages(const anna_mi_paged* h, const void* from, int64_t from_pages, void* to, int64_t to_pages,
               const std::vector<int32_t>& pairs, hipStream_t stream) {
  Copy c;
  c.from = (const uint8_t*)from;
  c.to = (uint8_t*)to;
  c.page = h->page_size();
  c.from_layer = from_pages * c.page;
  c.to_layer = to_pages * c.page;
  for (size_t at = 0; at < pairs.size(); at += UPDATE_WORDS) {
    c.pairs = (int32_t)std::min<size_t>(UPDATE_WORDS, pairs.size() - at) / 2;
    memcpy(c.words, pairs.data() + at, 8 * (size_t)c.pairs);
    const int rc = launch_copy(c, h->d.num_layers, stream);
    if (rc != ANNA_MI_OK) return rc;
  }
  return ANNA_MI_OK;
}

// Sequences in use, each at most once.
int check_seqs(anna_mi_paged* h, int64_t n, const int32_t* seqs) {
  int64_t k = 0;
  int rc = ANNA_MI_OK;
  for (; k < n; k++) {
    const int64_t s = seqs[k];
    if (s < 0 || s >= h->d.max_sequences || h->length[s] < 0) {
      set_error("sequence %lld is not in use", (long long)s);
      rc = ANNA_MI_EINVAL;
      break;
    }
    if (h->seen[s]) {
      set_error("sequence %lld appears twice", (long long)s);
      rc = ANNA_MI_EINVAL;
      break;
    }
    h->seen[s] = 1;
  }
  for (int64_t i = 0; i < k; i++) h->seen[seqs[i]] = 0;
  return rc;
}

// Gives back what sequence s holds from its page `from` on; the pages that nobody holds any more go to `freed`.
void drop_pages(anna_mi_paged* h, int64_t s, int64_t from, std::vector<int32_t>& freed) {
  int32_t* row = h->row(s);
  for (int64_t c = from; c < h->pages(s); c++) {
    if (--h->refs[row[c]] == 0) freed.push_back(row[c]);
    row[c] = 0;
  }
}

// On the stack so that they are taken again in the order in which they were freed.
void give_back(anna_mi_paged* h, const std::vector<int32_t>& freed) {
  h->free_pages.insert(h->free_pages.end(), freed.rbegin(), freed.rend());
}

// The layout of a span: its tiles, and the sizes that follow from them.  What a buffer has room for (the
// bounds) depends on the counts alone, so that a span can be filled again as its sequences grow.
struct Plan {
  std::vector<Record> records;
  int64_t few_rows = 16, tile_rows = 128, units = 0, unit_rows = 0, touches = 0, tokens = 0;
  int64_t items[2] = {0, 0}, bound[2] = {0, 0};  // of the split form, of the tile form
  int64_t touch_bound = 0, partial_rows = 0, partial_bound = 0;
  bool shared = false;  // a page with tokens of two sequences
};

// The fewest pages of an item of a form, `least` at least, with which there are at most `items` of them (or one a tile).
int64_t fewest_pages(const std::vector<Record>& records, int form, int64_t items, int64_t least) {
  int64_t low = least, high = least, tiles = 0;
  for (const Record& r : records)
    if (r.tiled == form) high = std::max<int64_t>(high, r.pages), tiles += r.pages > 0;
  items = std::max(items, tiles);
  while (low < high) {
    const int64_t mid = (low + high) / 2;
    int64_t n = 0;
    for (const Record& r : records)
      if (r.tiled == form) n += ceil_div(r.pages, mid);
    if (n <= items) high = mid;
    else low = mid + 1;
  }
  return low;
}

// starts null: of the tokens that an extend by counts is going to add.  The bounds are those of its span.
int make_plan(anna_mi_paged* h, int64_t n, const int32_t* seqs, const int64_t* starts, const int64_t* counts, Plan& p) {
  ANNA_CHECK(n >= 0 && (n == 0 || (seqs && counts)), "span: null arrays");
  int rc = check_seqs(h, n, seqs);
  if (rc != ANNA_MI_OK) return rc;
  const int64_t G = h->d.q_heads / h->d.kv_heads, H = h->d.kv_heads;
  const int64_t most = 4096 / h->d.head_dim;  // rows of a split tile whose sums stay in registers
  int64_t large = 0;                          // tiles of 256 rows
  std::vector<int32_t> held;                  // pages that others hold too
  std::vector<int64_t> ends;
  if (!starts) {
    for (int64_t i = 0; i < n; i++) {
      ends.push_back(h->length[seqs[i]]);
      ANNA_CHECK(counts[i] >= 0 && counts[i] <= h->d.max_pages * PAGE - ends[i], "span: %lld tokens more than the %lld of sequence %d, at most %lld fit",
                 (long long)counts[i], (long long)ends[i], (int)seqs[i], (long long)(h->d.max_pages * PAGE));
    }
  }
  const int64_t* const at = starts ? starts : ends.data();
  for (int64_t i = 0; i < n; i++) {
    ANNA_CHECK(!starts || (starts[i] >= 0 && counts[i] >= 0 && starts[i] <= h->length[seqs[i]] && counts[i] <= h->length[seqs[i]] - starts[i]),
               "span: tokens %lld .. %lld of sequence %d, which holds %lld", (long long)at[i],
               (long long)(at[i] + counts[i]), (int)seqs[i], (long long)h->length[seqs[i]]);
    p.tokens += counts[i];
    const int64_t rows = counts[i] * G;
    if (rows > TILE_LEAST) large += ceil_div(rows, 256);
    else p.few_rows = std::max(p.few_rows, std::min<int64_t>(most, rows > 32 ? 64 : rows > 16 ? 32 : 16));
  }
  ANNA_CHECK(p.tokens * G <= INT_MAX / 2, "span: too many tokens");
  // A wave takes 32 rows: workgroups of 8 share a page's conversion among twice as many rows as those of 4, which there
  // are twice as many of.  2048 tokens of 32 heads at the end of 32K: 1137 us, with 128 rows 1921 (at 64 dims 834 and 1065);
  // 12 prompts of 100 to 1500 tokens: 150 and 251 (106 and 117).
  if (large * H >= TILE_FILL && h->d.head_dim < 256) p.tile_rows = 256;
  int64_t offset = 0, tiles[2] = {0, 0}, rows_of[2] = {0, 0};  // tiles: those with tokens
  for (int64_t i = 0; i < n; i++) {
    const int64_t rows = counts[i] * G, f = rows > TILE_LEAST, R = f ? p.tile_rows : p.few_rows;
    for (int64_t t = 0; t < std::max<int64_t>(1, ceil_div(rows, R)); t++) {
      Record r = {};
      r.index = (int32_t)i, r.row = seqs[i], r.start = (int32_t)at[i], r.count = (int32_t)counts[i];
      r.offset = (int32_t)offset, r.tile = (int32_t)t, r.tiled = (int32_t)f;
      r.pages = rows ? (int32_t)((at[i] + (std::min(rows, (t + 1) * R) - 1) / G) / PAGE + 1) : 0;
      r.touch0 = (int32_t)p.touches;
      tiles[f] += rows > 0;
      rows_of[f] = std::max(rows_of[f], std::min(rows, R));
      p.records.push_back(r);
    }
    if (counts[i] > 0) {
      const int64_t first = at[i] / PAGE, last = (at[i] + counts[i] - 1) / PAGE;
      p.touches += last - first + 1;
      p.touch_bound += (counts[i] + PAGE - 2) / PAGE + 1;
      for (int64_t c = first; starts && c <= last; c++)
        if (h->refs[h->row(seqs[i])[c]] > 1) held.push_back(h->row(seqs[i])[c]);
    }
    offset += counts[i];
  }
  std::sort(held.begin(), held.end());
  p.shared = std::adjacent_find(held.begin(), held.end()) != held.end();
  // Tiles of the tile form in falling order of their pages, so that the long ones start first.
  if (tiles[1] > 1)
    std::stable_sort(p.records.begin(), p.records.end(), [](const Record& a, const Record& b) {
      return a.tiled != b.tiled ? a.tiled < b.tiled : a.tiled && a.pages > b.pages;
    });
  // How many pages an item takes: the workgroups of a launch shall fit the chip at once.
  const int64_t target[2] = {std::max<int64_t>(1, SPLIT_ONCE / H), std::max<int64_t>(1, TILE_ONCE / H)};
  const int64_t per[2] = {fewest_pages(p.records, 0, target[0], 1), fewest_pages(p.records, 1, target[1], TILE_PAGES)};
  for (Record& r : p.records) {
    const int f = r.tiled;
    const int64_t R = f ? p.tile_rows : p.few_rows, rows = std::min<int64_t>(R, r.count * G - r.tile * R);
    r.item0 = (int32_t)p.items[f];
    r.splits = (int32_t)ceil_div(r.pages, per[f]);
    r.part = -1;
    r.unit = -1;
    if (r.splits > 1) {
      r.part = (int32_t)p.partial_rows, r.unit = (int32_t)p.units++;
      p.partial_rows += r.splits * rows;
      p.unit_rows = std::max(p.unit_rows, rows);
    }
    p.items[f] += r.splits;
  }
  // a form has at most `target` items or one a tile; where there are more tiles, none is split
  for (int f = 0; f < 2; f++)
    if (rows_of[f] > 0) {
      p.bound[f] = std::max(target[f], tiles[f]);
      if (tiles[f] < target[f]) p.partial_bound += target[f] * rows_of[f];
    }
  ANNA_CHECK(p.partial_bound <= INT_MAX && H * std::max({p.bound[0], p.bound[1], p.touch_bound, (int64_t)p.records.size()}) <= MOST_GROUPS,
             "span: too many tokens");
  return ANNA_MI_OK;
}

template <class F> int guarded(anna_mi_paged* h, const char* what, F f) {
  ANNA_CHECK(h, "%s: null handle", what);
  try {
    std::lock_guard<std::mutex> g(h->lock);
    return f();
  } catch (const std::exception& e) {
    set_error("%s: %s", what, e.what());
    return ANNA_MI_EINVAL;
  }
}

}  // namespace

extern "C" {

int64_t anna_mi_sizeof_paged_desc(void) { return sizeof(anna_mi_paged_desc); }
int64_t anna_mi_sizeof_paged_span(void) { return sizeof(anna_mi_paged_span); }

int anna_mi_paged_create(const anna_mi_paged_desc* desc, anna_mi_paged** handle) {
  ANNA_CHECK(desc && handle, "paged_create: null argument");
  const anna_mi_paged_desc& d = *desc;
  ANNA_CHECK(d.dtype == ANNA_MI_BF16 || d.dtype == ANNA_MI_F16, "paged_create: dtype must be bf16 or fp16");
  ANNA_CHECK(d.head_dim == 64 || d.head_dim == 128 || d.head_dim == 256, "paged_create: head_dim must be 64, 128 or 256, got %lld",
             (long long)d.head_dim);
  ANNA_CHECK(d.kv_heads > 0 && d.kv_heads <= 1024 && d.q_heads > 0 && d.q_heads <= 65536 && d.q_heads % d.kv_heads == 0,
             "paged_create: q_heads must be a multiple of kv_heads");
  ANNA_CHECK(d.num_layers > 0 && d.num_layers <= 65535 && d.num_pages > 0 && d.num_pages < INT_MAX, "paged_create: bad num_layers or num_pages");
  ANNA_CHECK(d.max_sequences > 0 && d.max_pages > 0 && d.max_sequences <= INT_MAX / d.max_pages && d.max_pages <= INT_MAX / (2 * PAGE),
             "paged_create: bad max_sequences or max_pages");
  ANNA_CHECK(d.num_layers * ceil_div(d.kv_heads * page_bytes(d.head_dim), COPY_BYTES) <= MOST_GROUPS / 2,
             "paged_create: a page of all layers is too large");
  ANNA_CHECK(d.pool && d.table, "paged_create: null pool or table");
  ANNA_CHECK((uintptr_t)d.pool % 16 == 0, "paged_create: the pool must be 16-byte aligned");
  try {
    auto h = std::make_unique<anna_mi_paged>();
    h->d = d;
    h->table.assign(d.max_sequences * d.max_pages, 0);
    h->length.assign(d.max_sequences, -1);
    h->seen.assign(d.max_sequences, 0);
    h->refs.assign(d.num_pages, 0);
    for (int64_t i = d.num_pages - 1; i >= 0; i--) h->free_pages.push_back((int32_t)i);
    for (int64_t i = d.max_sequences - 1; i >= 0; i--) h->free_seqs.push_back((int32_t)i);
    *handle = h.release();
  } catch (const std::exception& e) {
    set_error("paged_create: %s", e.what());
    return ANNA_MI_EINVAL;
  }
  return ANNA_MI_OK;
}

int anna_mi_paged_destroy(anna_mi_paged* handle) {
  delete handle;
  return ANNA_MI_OK;
}

int anna_mi_paged_add(anna_mi_paged* h, int64_t n, int32_t* seqs) {
  return guarded(h, "paged_add", [&]() -> int {
    ANNA_CHECK(n >= 0 && (n == 0 || seqs), "paged_add: bad arguments");
    ANNA_CHECK(n <= (int64_t)h->free_seqs.size(), "paged_add: %lld sequences asked, %lld of %lld are free", (long long)n,
               (long long)h->free_seqs.size(), (long long)h->d.max_sequences);
    for (int64_t i = 0; i < n; i++) {
      seqs[i] = h->free_seqs.back();
      h->free_seqs.pop_back();
      h->length[seqs[i]] = 0;
    }
    return ANNA_MI_OK;
  });
}

int anna_mi_paged_fork(anna_mi_paged* h, int64_t n, const int32_t* parents, int32_t* children, void* stream) {
  return guarded(h, "paged_fork", [&]() -> int {
    ANNA_CHECK(n >= 0 && (n == 0 || (parents && children)), "paged_fork: bad arguments");
    for (int64_t i = 0; i < n; i++)
      ANNA_CHECK(parents[i] >= 0 && parents[i] < h->d.max_sequences && h->length[parents[i]] >= 0,
                 "paged_fork: sequence %d is not in use", (int)parents[i]);
    ANNA_CHECK(n <= (int64_t)h->free_seqs.size(), "paged_fork: %lld sequences asked, %lld of %lld are free", (long long)n,
               (long long)h->free_seqs.size(), (long long)h->d.max_sequences);
    const int rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    Updates up(h, stream);
    up.copies.reserve(3 * n);
    for (int64_t i = 0; i < n; i++) {
      const int32_t c = h->free_seqs.back(), p = parents[i];
      h->free_seqs.pop_back();
      children[i] = c;
      h->length[c] = h->length[p];
      const int64_t pages = h->pages(p);
      memcpy(h->row(c), h->row(p), 4 * pages);
      for (int64_t k = 0; k < pages; k++) h->refs[h->row(c)[k]]++;
      if (pages > 0) up.copy(c, p, pages);
    }
    return up.launch();
  });
}

int anna_mi_paged_extend(anna_mi_paged* h, int64_t n, const int32_t* seqs, const int64_t* counts, int64_t* starts, void* stream) {
  return guarded(h, "paged_extend", [&]() -> int {
    ANNA_CHECK(n >= 0 && (n == 0 || (seqs && counts)), "paged_extend: bad arguments");
    int rc = check_seqs(h, n, seqs);
    if (rc == ANNA_MI_OK) rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    // pages to take: those that are new, and a copy of a last page for all its holders but the last
    std::vector<int32_t> shared;  // last pages whose holders here each counted as one that leaves
    int64_t need = 0;
    for (int64_t i = 0; i < n; i++) {
      const int64_t old = h->length[seqs[i]];
      ANNA_CHECK(counts[i] >= 0, "paged_extend: count %lld", (long long)counts[i]);
      ANNA_CHECK(counts[i] <= h->d.max_pages * PAGE - old, "paged_extend: sequence %d would hold %lld tokens, at most %lld fit",
                 (int)seqs[i], (long long)(old + counts[i]), (long long)(h->d.max_pages * PAGE));
      need += ceil_div(old + counts[i], PAGE) - ceil_div(old, PAGE);
      if (counts[i] > 0 && old % PAGE != 0) {
        const int32_t last = h->row(seqs[i])[old / PAGE];
        if (h->refs[last] > 1) shared.push_back(last);
      }
    }
    if (!shared.empty()) {
      std::sort(shared.begin(), shared.end());
      for (size_t k = 0; k < shared.size();) {
        size_t e = k;
        while (e < shared.size() && shared[e] == shared[k]) e++;
        need += std::min<int64_t>(e - k, h->refs[shared[k]] - 1);
        k = e;
      }
    }
    ANNA_CHECK(need <= (int64_t)h->free_pages.size(), "paged_extend: %lld pages needed, %lld of %lld are free", (long long)need,
               (long long)h->free_pages.size(), (long long)h->d.num_pages);
    h->entries.reserve(2 * need);
    h->pairs.reserve(2 * shared.size());
    auto take = [&](int64_t seq, int64_t c) {
      const int32_t page = h->free_pages.back();
      h->free_pages.pop_back();
      h->refs[page] = 1;
      h->row(seq)[c] = page;
      h->entries.insert(h->entries.end(), {(int32_t)(seq * h->d.max_pages + c), page});
      return page;
    };
    for (int64_t i = 0; i < n; i++) {
      const int64_t s = seqs[i], old = h->length[s];
      if (starts) starts[i] = old;
      if (counts[i] == 0) continue;
      if (old % PAGE != 0) {
        const int32_t last = h->row(s)[old / PAGE];
        if (h->refs[last] > 1) {
          h->refs[last]--;
          const int32_t page = take(s, old / PAGE);
          h->pairs.insert(h->pairs.end(), {last, page});
        }
      }
      for (int64_t c = ceil_div(old, PAGE); c < ceil_div(old + counts[i], PAGE); c++) take(s, c);
      h->length[s] = old + counts[i];
    }
    return ANNA_MI_OK;
  });
}

int anna_mi_paged_truncate(anna_mi_paged* h, int32_t seq, int64_t length, void* stream) {
  return guarded(h, "paged_truncate", [&]() -> int {
    int rc = check_seqs(h, 1, &seq);
    if (rc != ANNA_MI_OK) return rc;
    ANNA_CHECK(length >= 0 && length <= h->length[seq], "paged_truncate: length %lld of a sequence of %lld", (long long)length,
               (long long)h->length[seq]);
    rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    std::vector<int32_t> freed;
    const int64_t keep = ceil_div(length, PAGE);
    Updates up(h, stream);
    if (keep < h->pages(seq)) up.copy(seq, -1, keep);
    drop_pages(h, seq, keep, freed);
    give_back(h, freed);
    h->length[seq] = length;
    return up.launch();
  });
}

int anna_mi_paged_free(anna_mi_paged* h, int64_t n, const int32_t* seqs, void* stream) {
  return guarded(h, "paged_free", [&]() -> int {
    ANNA_CHECK(n >= 0 && (n == 0 || seqs), "paged_free: bad arguments");
    int rc = check_seqs(h, n, seqs);
    if (rc == ANNA_MI_OK) rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    Updates up(h, stream);
    std::vector<int32_t> freed;
    for (int64_t i = 0; i < n; i++) {
      if (h->length[seqs[i]] > 0) up.copy(seqs[i], -1, 0);
      drop_pages(h, seqs[i], 0, freed);
      h->length[seqs[i]] = -1;
    }
    give_back(h, freed);
    for (int64_t i = n - 1; i >= 0; i--) h->free_seqs.push_back(seqs[i]);
    return up.launch();
  });
}

int anna_mi_paged_compact(anna_mi_paged* h, int64_t* live, void* stream) {
  return guarded(h, "paged_compact", [&]() -> int {
    int rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    const int64_t n = h->d.num_pages - (int64_t)h->free_pages.size();
    // pages behind the first n move into the holes before them: sources and targets are disjoint
    std::vector<int32_t> to(h->d.num_pages, -1), pairs;
    int64_t hole = 0;
    for (int64_t p = n; p < h->d.num_pages; p++) {
      if (h->refs[p] == 0) continue;
      while (h->refs[hole] != 0) hole++;
      pairs.insert(pairs.end(), {(int32_t)p, (int32_t)hole});
      to[p] = (int32_t)hole++;
    }
    Updates up(h, stream);
    for (int64_t s = 0; s < h->d.max_sequences; s++)
      for (int64_t c = 0; h->length[s] > 0 && c < h->pages(s); c++) {
        int32_t& page = h->row(s)[c];
        if (to[page] < 0) continue;
        page = to[page];
        up.entry(s * h->d.max_pages + c, page);
      }
    for (size_t k = 0; k < pairs.size(); k += 2) std::swap(h->refs[pairs[k]], h->refs[pairs[k + 1]]);
    h->free_pages.clear();
    for (int64_t p = h->d.num_pages - 1; p >= n; p--) h->free_pages.push_back((int32_t)p);
    if (live) *live = n;
    rc = copy_pages(h, h->d.pool, h->d.num_pages, h->d.pool, h->d.num_pages, pairs, as_stream(stream));
    return rc != ANNA_MI_OK ? rc : up.launch();
  });
}

int anna_mi_paged_resize(anna_mi_paged* h, int64_t num_pages, void* pool, void* stream) {
  return guarded(h, "paged_resize", [&]() -> int {
    const int64_t n = h->d.num_pages - (int64_t)h->free_pages.size();
    ANNA_CHECK(num_pages >= n && num_pages > 0 && num_pages < INT_MAX, "paged_resize: %lld pages, %lld are in use", (long long)num_pages,
               (long long)n);
    ANNA_CHECK(pool && (uintptr_t)pool % 16 == 0 && pool != h->d.pool, "paged_resize: needs another, 16-byte aligned pool");
    int rc = flush(h, stream);
    if (rc != ANNA_MI_OK) return rc;
    std::vector<int32_t> to(h->d.num_pages, -1), pairs, refs(num_pages, 0);
    pairs.reserve(2 * num_pages);
    int32_t next = 0;
    Updates up(h, stream);
    for (int64_t s = 0; s < h->d.max_sequences; s++)
      for (int64_t c = 0; h->length[s] > 0 && c < h->pages(s); c++) {
        int32_t& page = h->row(s)[c];
        if (to[page] < 0) {
          to[page] = next;
          refs[next] = h->refs[page];
          pairs.insert(pairs.end(), {page, next++});
        }
        if (page != to[page]) up.entry(s * h->d.max_pages + c, to[page]);
        page = to[page];
      }
    for (int64_t p = next; p < num_pages; p++) pairs.insert(pairs.end(), {-1, (int32_t)p});
    const void* old = h->d.pool;
    const int64_t old_pages = h->d.num_pages;
    h->refs.swap(refs);
    h->free_pages.clear();
    for (int64_t p = num_pages - 1; p >= next; p--) h->free_pages.push_back((int32_t)p);
    h->d.pool = pool;
    h->d.num_pages = num_pages;
    rc = copy_pages(h, old, old_pages, pool, num_pages, pairs, as_stream(stream));
    return rc != ANNA_MI_OK ? rc : up.launch();
  });
}

int anna_mi_paged_lengths(anna_mi_paged* h, int64_t n, const int32_t* seqs, int64_t* lengths, int64_t* live_pages) {
  return guarded(h, "paged_lengths", [&]() -> int {
    ANNA_CHECK(n >= 0 && (n == 0 || (seqs && lengths)), "paged_lengths: bad arguments");
    for (int64_t i = 0; i < n; i++)
      lengths[i] = seqs[i] >= 0 && seqs[i] < h->d.max_sequences ? h->length[seqs[i]] : -1;
    if (live_pages) *live_pages = h->d.num_pages - (int64_t)h->free_pages.size();
    return ANNA_MI_OK;
  });
}

int anna_mi_paged_span_plan(anna_mi_paged* h, int64_t n, const int32_t* seqs, const int64_t* starts, const int64_t* counts,
                            anna_mi_paged_span* span) {
  return guarded(h, "paged_span_plan", [&]() -> int {
    ANNA_CHECK(span, "paged_span_plan: null span");
    Plan p;
    const int rc = make_plan(h, n, seqs, starts, counts, p);
    if (rc != ANNA_MI_OK) return rc;
    memset(span, 0, sizeof(*span));
    span->sequences = n;
    span->tokens = p.tokens;
    span->few_rows = p.few_rows;
    span->tile_rows = p.tile_rows;
    span->split_capacity = p.bound[0];
    span->unit_capacity = (int64_t)p.records.size();
    span->touch_capacity = p.touch_bound;
    span->tile_capacity = p.bound[1];
    span->partial_rows = p.partial_bound;
    span->words = sections(*span).words;
    return ANNA_MI_OK;
  });
}

int anna_mi_paged_span_fill(anna_mi_paged* h, int64_t n, const int32_t* seqs, const int64_t* starts, const int64_t* counts,
                            anna_mi_paged_span* span, void* stream) {
  return guarded(h, "paged_span_fill", [&]() -> int {
    ANNA_CHECK(span && span->buf && (uintptr_t)span->buf % 16 == 0, "paged_span_fill: null or unaligned buffer");
    ANNA_CHECK(n <= 0 || starts, "paged_span_fill: null starts");
    Plan p;
    const int rc = make_plan(h, n, seqs, starts, counts, p);
    if (rc != ANNA_MI_OK) return rc;
    ANNA_CHECK(n == span->sequences && p.tokens == span->tokens && p.few_rows == span->few_rows && p.tile_rows == span->tile_rows &&
                   p.items[0] <= span->split_capacity && p.items[1] <= span->tile_capacity && (int64_t)p.records.size() <= span->unit_capacity &&
                   p.touches <= span->touch_capacity && p.partial_rows <= span->partial_rows && sections(*span).words <= span->words,
               "span: these tokens do not fit the span that is filled");
    ANNA_CHECK(p.partial_rows == 0 || (span->partial_stats && span->partial_values), "paged_span_fill: null partials");
    ANNA_CHECK(!p.shared || !span->stored, "span: two sequences share a page that a captured store of this span would write");
    span->shared = p.shared;
    span->split_items = p.items[0];
    span->tile_items = p.items[1];
    span->split_units = p.units;
    span->split_rows = p.unit_rows;
    span->touch_items = p.touches;
    Updates up(h, stream);
    const Sections at = sections(*span);
    Update& u = up.u;
    u.buf = span->buf;
    u.header[0] = (int32_t)p.items[0], u.header[1] = (int32_t)p.items[1], u.header[2] = (int32_t)p.units;
    u.header[3] = (int32_t)p.touches;
    u.rows_at = at.rows, u.split_at = at.split, u.tile_at = at.tile, u.units_at = at.units, u.touch_at = at.touch;
    u.group = (int32_t)(h->d.q_heads / h->d.kv_heads);
    u.split_rows = (int32_t)p.few_rows;
    u.tile_rows = (int32_t)p.tile_rows;
    up.records.resize(p.records.size() * (sizeof(Record) / 4));
    if (!p.records.empty()) memcpy(up.records.data(), p.records.data(), p.records.size() * sizeof(Record));
    up.entries.swap(h->entries);
    up.pairs.swap(h->pairs);
    return up.launch();
  });
}

namespace {
int check_layer(anna_mi_paged* h, int64_t layer, const anna_mi_paged_span* span, const char* what) {
  ANNA_CHECK(span && span->buf, "%s: null span", what);
  ANNA_CHECK(layer >= 0 && layer < h->d.num_layers, "%s: layer %lld of %lld", what, (long long)layer, (long long)h->d.num_layers);
  return ANNA_MI_OK;
}
uint8_t* layer_pool(anna_mi_paged* h, int64_t layer) {
  return (uint8_t*)h->d.pool + layer * h->d.num_pages * h->page_size();
}
bool aligned(const void* p, int64_t token, int64_t head) { return (uintptr_t)p % 16 == 0 && token % 8 == 0 && head % 8 == 0; }
}  // namespace

int anna_mi_paged_store(anna_mi_paged* h, int64_t layer, anna_mi_paged_span* span, const void* keys, int64_t key_stride_token,
                        int64_t key_stride_head, const void* values, int64_t value_stride_token, int64_t value_stride_head,
                        int capacity_grid, void* stream) {
  return guarded(h, "paged_store", [&]() -> int {
    int rc = check_layer(h, layer, span, "paged_store");
    if (rc == ANNA_MI_OK) rc = flush(h, stream);
    if (rc != ANNA_MI_OK || span->tokens == 0) return rc;
    ANNA_CHECK(!span->shared, "paged_store: two sequences of the span share a page");
    ANNA_CHECK(keys && values, "paged_store: null keys or values");
    ANNA_CHECK(aligned(keys, key_stride_token, key_stride_head) && aligned(values, value_stride_token, value_stride_head),
               "paged_store: keys and values need rows of 16-byte alignment");
    if (capacity_grid) span->stored = 1;
    return launch_store(h->d.dtype, h->d.head_dim, layer_pool(h, layer), h->d.table, h->d.max_pages, span->buf,
                        (const Touch*)(span->buf + sections(*span).touch),
                        capacity_grid ? span->touch_capacity : span->touch_items, h->d.kv_heads, keys, key_stride_token,
                        key_stride_head, values, value_stride_token, value_stride_head, as_stream(stream));
  });
}

int anna_mi_paged_read(anna_mi_paged* h, int64_t layer, const anna_mi_paged_span* span, void* keys, void* values, int capacity_grid,
                       void* stream) {
  return guarded(h, "paged_read", [&]() -> int {
    int rc = check_layer(h, layer, span, "paged_read");
    if (rc == ANNA_MI_OK) rc = flush(h, stream);
    if (rc != ANNA_MI_OK || span->tokens == 0) return rc;
    ANNA_CHECK(keys && values && (uintptr_t)keys % 16 == 0 && (uintptr_t)values % 16 == 0, "paged_read: null or unaligned output");
    return launch_read(h->d.dtype, h->d.head_dim, layer_pool(h, layer), h->d.table, h->d.max_pages, span->buf,
                       (const Touch*)(span->buf + sections(*span).touch),
                       capacity_grid ? span->touch_capacity : span->touch_items, h->d.kv_heads, keys, values,
                       as_stream(stream));
  });
}

int anna_mi_paged_attend(anna_mi_paged* h, int64_t layer, const anna_mi_paged_span* span, const void* query,
                         int64_t query_stride_token, int64_t query_stride_head, const void* gate, int64_t gate_stride_token,
                         int64_t gate_stride_head, void* out, float scaling, int capacity_grid, void* stream) {
  return guarded(h, "paged_attend", [&]() -> int {
    int rc = check_layer(h, layer, span, "paged_attend");
    if (rc == ANNA_MI_OK) rc = flush(h, stream);
    if (rc != ANNA_MI_OK || span->tokens == 0) return rc;
    ANNA_CHECK(query && out && (uintptr_t)out % 16 == 0, "paged_attend: null query or output, or an unaligned output");
    ANNA_CHECK(aligned(query, query_stride_token, query_stride_head) &&
                   (!gate || aligned(gate, gate_stride_token, gate_stride_head)),
               "paged_attend: query and gate need rows of 16-byte alignment");
    ANNA_CHECK(scaling > 0 && scaling < 1.0e30f, "paged_attend: scaling must be positive and finite");
    const Sections at = sections(*span);
    Attend a;
    a.pool = layer_pool(h, layer);
    a.table = h->d.table;
    a.width = h->d.max_pages;
    a.header = span->buf;
    a.split = (const Item*)(span->buf + at.split);
    a.tile = (const Item*)(span->buf + at.tile);
    a.units = (const Unit*)(span->buf + at.units);
    a.query = query, a.q_token = query_stride_token, a.q_head = query_stride_head;
    a.gate = gate, a.g_token = gate_stride_token, a.g_head = gate_stride_head;
    a.out = out;
    a.stats = span->partial_stats, a.values = span->partial_values;
    a.scale = scaling * 1.44269504088896340736f;
    a.kv_heads = (int32_t)h->d.kv_heads;
    a.group = (int32_t)(h->d.q_heads / h->d.kv_heads);
    Grid g = {span->split_items, span->few_rows, span->tile_items, span->tile_rows, span->split_units, span->split_rows};
    if (capacity_grid) {
      g.split_items = span->split_capacity, g.tile_items = span->tile_capacity, g.units = span->unit_capacity;
      g.unit_rows = span->tile_capacity > 0 ? span->tile_rows : span->few_rows;
    }
    return launch_attend(h->d.dtype, h->d.head_dim, a, g, as_stream(stream));
  });
}

}  // extern "C"
