// What the paged 4-bit cache's host side and kernels share: the page layout (anna_mi.h), the span's
// buffer and the launches.
#pragma once

#include "common.hpp"

namespace anna {
namespace paged {

constexpr int PAGE = 64;   // tokens of a page
constexpr int GROUP = 64;  // values with one scale and zero
constexpr int COPY_BYTES = 16384;  // of a page of all KV heads that a workgroup copies
// What codes carry when they enter a matrix instruction, and offsets are without: 16 + code is exact in bf16's
// eight bits by bit operations alone, and the smallest such number keeps the sums that cancel small.
constexpr int CODE_BASE = 16;

// Byte offsets in a page of one KV head of head_dim D.
constexpr int64_t page_bytes(int64_t D) { return 72 * D; }
constexpr int V_CODES = 32, K_SCALES = 64, K_OFFSETS = 66, V_SCALES = 68, V_OFFSETS = 70;  // times D

// A tile's share of a sequence's pages: one workgroup of an attention launch for every KV head.
struct Item {
  int32_t row;     // page table row
  int32_t start;   // position of the span's first token of this sequence
  int32_t count;   // its tokens
  int32_t offset;  // and where they stand in the packed queries
  int32_t page0, page1;
  int32_t part;  // first row of its partial results; -1: it is its tile's only item
  int32_t tile;  // query rows tile * R ..: row r is token r / G, query head r % G of the KV head
};
// A tile that several items share: the merge's work.
struct Unit {
  int32_t offset, row0, rows, part, splits, pad[3];
};
// The tokens of a span in one page.
struct Touch {
  int32_t row, page, begin, end, token, pad[3];
};

// Where the sections of a span's buffer stand, in words: header, table rows, items, units, touches.
struct Sections {
  int64_t rows, split, tile, units, touch, words;
};
constexpr int HEADER = 8;  // split items, tile items, units, touches
inline Sections sections(const anna_mi_paged_span& s) {
  auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  Sections o;
  o.rows = HEADER;
  o.split = o.rows + up(s.sequences);
  o.tile = o.split + 8 * s.split_capacity;
  o.units = o.tile + 8 * s.tile_capacity;
  o.touch = o.units + 8 * s.unit_capacity;
  o.words = o.touch + 8 * s.touch_capacity;
  return o;
}

// One tile of one sequence, from which its items, its unit and (tile 0) its touches are written.
struct Record {
  int32_t index, row, start, count, offset, tile, item0, pages, splits, part, unit, touch0;
  int32_t tiled;  // 1: of the tile form
};

// The words of an update travel in the kernel's arguments (at most 4 KB of them): no staging memory whose
// life would have to be tied to the stream, and one launch for the few words of a decode step.
constexpr int UPDATE_WORDS = 952;
struct Update {
  int32_t* table;
  int64_t width;
  int32_t* buf;  // of the span whose records these are
  int32_t header[4];
  int64_t rows_at, split_at, tile_at, units_at, touch_at;
  int32_t group, split_rows, tile_rows;  // query heads of a KV head; rows of the two forms' tiles
  uint8_t* pool;  // for page copies within it: bytes of a layer and of a page of all KV heads, layers
  int64_t pool_layer, page;
  int32_t layers;
  int32_t records, entries, copies, pairs;  // in this order in words
  int32_t words[UPDATE_WORDS];  // Record; (index, page); (row, source row or -1, pages): the rest of row is zeroed; (page, page)
};
static_assert(sizeof(Update) <= 4096, "an update is a kernel argument");
int launch_update(const Update& u, hipStream_t stream);

struct Copy {
  const uint8_t* from;
  uint8_t* to;
  int64_t from_layer, to_layer;  // bytes of a layer
  int64_t page;                  // bytes of a page of all KV heads
  int32_t pairs;
  int32_t words[UPDATE_WORDS];  // (source page or -1 for zeros, page)
};
static_assert(sizeof(Copy) <= 4096, "a copy is a kernel argument");
int launch_copy(const Copy& c, int64_t layers, hipStream_t stream);

struct Attend {
  const uint8_t* pool;  // of the layer
  const int32_t* table;
  int64_t width;
  const int32_t* header;
  const Item *split, *tile;
  const Unit* units;
  const void *query, *gate;
  int64_t q_token, q_head, g_token, g_head;
  void* out;
  float* stats;
  float* values;
  float scale;  // scaling * log2(e)
  int32_t kv_heads, group;
};
struct Grid {
  int64_t split_items, few_rows, tile_items, tile_rows, units, unit_rows;
};
int launch_attend(int dtype, int64_t head_dim, const Attend& a, const Grid& g, hipStream_t stream);
int launch_store(int dtype, int64_t head_dim, uint8_t* pool, const int32_t* table, int64_t width,
                 const int32_t* header, const Touch* touch, int64_t touches, int64_t kv_heads, const void* keys, int64_t k_token, int64_t k_head, const void* values,
                 int64_t v_token, int64_t v_head, hipStream_t stream);
int launch_read(int dtype, int64_t head_dim, const uint8_t* pool, const int32_t* table, int64_t width,
                const int32_t* header, const Touch* touch, int64_t touches, int64_t kv_heads, void* keys, void* values, hipStream_t stream);

}  // namespace paged
}  // namespace anna
