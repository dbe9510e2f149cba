// Work plan of the attention over the paged cache: built on the host
// (paged_plan.cpp), read by the kernels.
//
// A unit is (request, kv head, row tile): consecutive query rows of one kv head,
// row = token * G + g. A unit's visible keys are cut into spans of whole 128-key
// tiles; an item is one span. A unit of one item is written out directly; the
// items of a split unit leave partial states in consecutive slots, and the CTA
// that finishes last (one ticket per split unit) joins them in slot order, so the
// result does not depend on which one that is.
#pragma once

#include <stdint.h>

namespace d2sd {
namespace paged {

constexpr int kTileKeys = 128;
constexpr int kRowsTile = 16;    // query rows of a unit of the rows kernel
constexpr int kRowsLimit = 16;   // requests of more rows per kv head go to the tiles kernel
constexpr int kMagic = 0x50474131;

// header: magic, then one section per kernel (S_*), kSectionInts ints each
enum { H_MAGIC = 0, H_REQUESTS, H_TOKENS, H_GROUP, H_KV_HEADS, H_SECTION, };
enum { S_CTAS = 0, S_ITEMS, S_SLOTS, S_TICKETS, S_OFF_CTA, S_OFF_ITEMS, kSectionInts };
constexpr int kSections = 2;  // 0: rows kernel, 1: tiles kernel
constexpr int kHeaderInts = 32;

enum {
  P_REQ = 0,
  P_HEAD,
  P_TOK0,      // q row of the request's first token
  P_ROW0,      // first row of the unit, inside the request
  P_NROWS,     // rows of the unit
  P_KEY0,      // span [key0, key1): multiples of 128, key1 cut at the last visible key
  P_KEY1,
  P_POS0,      // position of the request's token 0 (non-causal: kNoLimit)
  P_WINDOW,    // 0: none
  P_PAGE_OFF,  // the request's first entry in the page table
  P_KV_LEN,
  P_SLOT,        // this item's slot, -1: the unit's only item
  P_FIRST_SLOT,  // of the unit
  P_PARTS,
  P_TICKET,
  P_PAD,
  kItemInts
};
constexpr int kNoLimit = 1 << 30;

// Workspace: tickets of the rows units (2 per CTA: a CTA's first and last item can
// be spans of split units) and of the tiles units (one for each of two q tiles),
// then the slots in the same order.
constexpr int64_t tile_tickets_at(int num_ctas) { return 2 * static_cast<int64_t>(num_ctas); }
constexpr int64_t ticket_bytes(int num_ctas) { return (6 * 4 * static_cast<int64_t>(num_ctas) + 127) / 128 * 128; }
constexpr int64_t rows_slot_floats(int head_dim) { return kRowsTile * (head_dim + 2); }
constexpr int64_t tile_slot_floats(int head_dim) { return 128 * (head_dim + 2); }
constexpr int64_t tile_slots_at(int num_ctas, int head_dim) {  // floats behind the first slot
  return 2 * static_cast<int64_t>(num_ctas) * rows_slot_floats(head_dim);
}
constexpr int64_t workspace_bytes(int num_ctas, int head_dim) {
  return ticket_bytes(num_ctas) +
         4 * (tile_slots_at(num_ctas, head_dim) + 4 * static_cast<int64_t>(num_ctas) * tile_slot_floats(head_dim));
}

}  // namespace paged
}  // namespace d2sd
