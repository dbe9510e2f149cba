// Work plan of the attention over the paged cache: built on the host
// (paged_plan.cpp), read by the kernels.
//
// A unit is (request, kv head, row tile): consecutive query rows of one kv head,
// row = token * G + g. A unit's visible keys, from the first one's page of 16 on, are
// cut into spans of whole 128-key tiles; an item is one span. A unit of one item is written out directly; the
// items of a split unit leave partial states in consecutive slots, which a second
// kernel joins in slot order (kept apart so that all SMs join, and no state stays
// behind in the workspace), 4 or 8 rows to an entry of the join list. Where every unit
// can have a cluster of CTAs of its own (few units, not too many keys), its spans are
// joined inside the cluster instead: parts > 1 and no join list.
#pragma once

#include <stdint.h>

namespace d2sd {
namespace paged {

constexpr int kTileKeys = 128;
constexpr int kRowsTile = 16;    // query rows of a unit of the rows kernel
constexpr int kRowsCtas = 4;     // CTAs of the rows kernel on an SM
// Requests of more rows per kv head go to the tiles kernel. Measured with 16 requests
// of 2k to 16k keys, there and in tiles of 16 rows of the rows kernel. 32 / 8 heads of
// 128: 16-bit, 20 rows 122 us and 194; 8-bit, 20 rows 199 and 131, 32 rows 198 and 132, 64
// rows 198 and 240. Heads of 64 (32 or 64 query heads): 16-bit, 24 to 32 rows 115 and 100,
// 40 rows 117 and 133; 8-bit, 32 rows 160 and 98, 40 rows 163 and 136, 64 rows 163 and 178.
// One limit for both head sizes, so heads of 64 give away 15 us at 17 to 32 rows of 16-bit
// pages.
constexpr int kRowsLimit = 16, kRowsLimit8 = 32;
constexpr int kCluster = 8;  // CTAs of a cluster at most
constexpr int kMagic = 0x50474131;

// header: magic, then one section per kernel (S_*), kSectionInts ints each
enum { H_MAGIC = 0, H_REQUESTS, H_TOKENS, H_GROUP, H_KV_HEADS, H_SECTION, };
enum { S_CTAS = 0, S_ITEMS, S_SLOTS, S_JOINS, S_OFF_CTA, S_OFF_ITEMS, S_OFF_JOINS, S_PARTS, kSectionInts };  // S_PARTS: most spans of a unit
constexpr int kSections = 2;  // 0: rows kernel, 1: tiles kernel
constexpr int kHeaderInts = 32;

enum {
  P_REQ = 0,
  P_HEAD,
  P_TOK0,      // q row of the request's first token
  P_ROW0,      // first row of the unit, inside the request
  P_NROWS,     // rows of the unit
  P_KEY0,      // span [key0, key1): from a page's first key, whole tiles up to the last one
  P_KEY1,
  P_POS0,      // position of the request's token 0 (non-causal: kNoLimit)
  P_WINDOW,    // 0: none
  P_PAGE_OFF,  // the request's first entry in the page table
  P_KV_LEN,
  P_SLOT,         // this item's slot, -1: the unit's only item
  P_PARTS,        // items of the unit
  P_FIRST_TOKEN,  // of the unit, inside the request (P_ROW0 / G)
  P_PAD0,
  P_PAD1,
  kItemInts
};
constexpr int kNoLimit = 1 << 30;

// Entry of a join list: rows J_ROW0 .. of one q tile (tiles: slots 2 * slot + tile).
enum {
  J_SLOT = 0,  // the unit's first slot (tiles: of this q tile)
  J_STEP,      // slots from one part to the next
  J_PARTS,
  J_SLOT_ROW,  // first row inside the slot
  J_ROWS,      // rows of the entry
  J_ROW0,      // first row inside the request
  J_TOK0,      // q row of the request's first token
  J_HEAD,
  kJoinInts
};
constexpr int kJoinRows[kSections] = {4, 8};

// A slot holds [head_dim / 4][rows] of four columns each, then the rows' m and l.
// A CTA's first and last item can be spans of split units, so 2 slots per CTA do
// (tiles: 4, one for each q tile). Workspace: the rows slots, then the tiles slots.
constexpr int section_ctas(int section, int num_ctas) { return section == 0 ? kRowsCtas * num_ctas : num_ctas; }
constexpr int64_t rows_slot_floats(int head_dim) { return kRowsTile * (head_dim + 2); }
constexpr int64_t tile_slot_floats(int head_dim) { return 128 * (head_dim + 2); }
constexpr int64_t tile_slots_at(int num_ctas, int head_dim) {  // floats
  return 2 * static_cast<int64_t>(section_ctas(0, num_ctas)) * rows_slot_floats(head_dim);
}
constexpr int64_t workspace_bytes(int num_ctas, int head_dim) {
  return 4 * (tile_slots_at(num_ctas, head_dim) + 4 * static_cast<int64_t>(num_ctas) * tile_slot_floats(head_dim));
}

}  // namespace paged
}  // namespace d2sd
