// Host-side plan of the attention over the paged cache (paged_plan.h).
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <functional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/d2sd.h"
#include "paged_plan.h"

namespace d2sd {
void set_last_error(const std::string& msg);

namespace {
using namespace paged;

int plan_fail(int code, const char* msg) {
  set_last_error(std::string("d2sd_paged_plan: ") + msg);
  return code;
}

struct Unit {
  int32_t req, head, tok0, row0, nrows, key0, key1, pos0, page_off, kv_len;
  int32_t weight;  // cost of a tile
  int32_t tiles() const { return key1 > key0 ? (key1 - key0 + kTileKeys - 1) / kTileKeys : 0; }
};

// Whole units on the CTAs, the costliest first and each on the CTA with the least so
// far, if that leaves no CTA with more above its share than cutting and joining would
// cost: two starts of an item, or a sixty-fourth. Then nothing has to be joined. Measured,
// whole and cut: a prompt of 8192 tokens 480 us and 516; 40 chunks of 100 to 900 tokens
// 587 and 651; 300 single tokens over 100 to 2000 keys 205 and 220. first: the first item
// of each CTA.
bool place_whole(const std::vector<Unit>& units, int ctas, int extra, int32_t group, int32_t window,
                 std::vector<int32_t>& items, std::vector<int32_t>& first) {
  const size_t n = static_cast<size_t>(ctas);
  if (units.size() < n) return false;
  int64_t total = 0, fixed = 0, most = 0;
  for (const Unit& u : units) {
    const int64_t cost = static_cast<int64_t>(u.tiles() + extra) * u.weight;
    total += cost;
    most = std::max(most, cost);
    fixed = std::max(fixed, static_cast<int64_t>(extra) * u.weight);
  }
  const int64_t share = total / static_cast<int64_t>(n), limit = share + std::max(2 * fixed, share / 64);
  if (most > limit) return false;
  std::vector<uint64_t> order;  // costliest first, then in order
  order.reserve(units.size());
  for (size_t i = 0; i < units.size(); ++i) {
    const uint64_t cost = static_cast<uint64_t>(units[i].tiles() + extra) * units[i].weight;
    order.push_back((~cost << 32) | i);
  }
  std::sort(order.begin(), order.end());
  std::vector<std::pair<int64_t, int32_t>> heap;  // (load, CTA), least load first
  for (size_t c = 0; c < n; ++c) heap.push_back({0, static_cast<int32_t>(c)});
  const auto later = std::greater<std::pair<int64_t, int32_t>>();
  std::vector<int32_t> cta(units.size());
  first.assign(n + 1, 0);
  for (uint64_t key : order) {
    const size_t i = static_cast<uint32_t>(key);
    std::pop_heap(heap.begin(), heap.end(), later);
    auto& least = heap.back();
    least.first += static_cast<int64_t>(units[i].tiles() + extra) * units[i].weight;
    if (least.first > limit) return false;
    cta[i] = least.second;
    ++first[least.second + 1];
    std::push_heap(heap.begin(), heap.end(), later);
  }
  for (size_t c = 0; c < n; ++c) first[c + 1] += first[c];
  std::vector<int32_t> next(first.begin(), first.end() - 1);
  items.resize(units.size() * kItemInts);
  for (uint64_t key : order) {
    const size_t i = static_cast<uint32_t>(key);
    const Unit& u = units[i];
    const int32_t it[kItemInts] = {u.req,  u.head,     u.tok0,   u.row0, u.nrows, u.key0, u.key1, u.pos0,
                                   window, u.page_off, u.kv_len, -1,     1,       u.row0 / group, 0, 0};
    memcpy(items.data() + static_cast<size_t>(next[cta[i]]++) * kItemInts, it, sizeof(it));
  }
  return true;
}

// Few units of the rows kernel: a cluster of 8, 4 or 2 CTAs for each, its pages shared
// out evenly, if that ends before the same units cut over all CTAs and joined by a second
// kernel would. Both estimates in units of a CTA's time for 128 keys with the memory to
// itself (2.5 us in 16 bits, 1.9 us in 8): all CTAs at once take 2.4 (1.9) times that, and
// the join costs 4 (5) of them. Measured, clusters against the cut, 8 kv heads of 128, one
// new token each in 16 bits: 1 request of 1000 keys 9.2 us and 15.4, of 8000 25 and 20; 9
// of 1000 14.3 and 21.5; 18 of 2000 32 and 40; 37 of 500 18.2 and 23.3. The choice was
// within 1 us of the better one in all of 48 such pairs at heads of 128 and of 64, 16- and
// 8-bit (heads of 64, 16-bit: 8.7 and 14.3, 23 and 17, 11.5 and 17.9, 23.6 and 24.1, 12.8
// and 18.4).
bool place_clusters(const std::vector<Unit>& units, int ctas, int32_t group, int32_t window, bool eight_bit,
                    std::vector<int32_t>& items, std::vector<int32_t>& first, int32_t* parts) {
  int32_t most = 0, size = kCluster;
  int64_t tiles = 0;
  for (const Unit& u : units) most = std::max(most, u.key1 - u.key0), tiles += u.tiles();
  // up to half of the CTAs, or pairs on all of them
  while (size > 2 && units.size() * size * 2 > static_cast<size_t>(ctas)) size /= 2;
  if (units.size() * size > static_cast<size_t>(ctas) || most <= kTileKeys) return false;
  const double full = eight_bit ? 1.9 : 2.4, join = eight_bit ? 5 : 4;
  const double span = (most + size - 1) / size / static_cast<double>(kTileKeys) * (eight_bit ? 1.25 : 1);
  const double load = static_cast<double>(tiles) / ctas, used = units.size() * size / static_cast<double>(ctas);
  if (span * std::max(1., full * used) > std::max(1., load) * std::max(1., full * std::min(1., load)) + join) return false;
  *parts = size;
  first.assign(1, 0);
  for (const Unit& u : units) {
    const int32_t pages = (u.key1 - u.key0 + 15) / 16, per = (pages + size - 1) / size * 16;
    for (int32_t p = 0; p < size; ++p) {
      const int32_t k0 = std::min(u.key0 + p * per, u.key1), k1 = std::min(k0 + per, u.key1);
      const int32_t it[kItemInts] = {u.req,  u.head,     u.tok0,   u.row0, u.nrows,  k0, k1, u.pos0,
                                     window, u.page_off, u.kv_len, -1,     size,     u.row0 / group, 0, 0};
      items.insert(items.end(), it, it + kItemInts);
      first.push_back(static_cast<int32_t>(items.size() / kItemInts));
    }
  }
  return true;
}

// The units in order, cut where a CTA's share of the cost ends. An item costs its
// tiles and `extra` more (its start, its end and, for a split unit, the joining),
// each of the unit's weight, so a CTA of many small items gets fewer tiles.
void cut(const std::vector<Unit>& units, int ctas, int section, int32_t group, int32_t window, int32_t flags,
         std::vector<int32_t>& items, std::vector<int32_t>& first, std::vector<int32_t>& joins, int32_t* slots, int32_t* most) {
  const int extra = section == 0 ? 1 : 4;
  const int q_tile = section == 0 ? kRowsTile : 128 / group * group, per = section == 0 ? 1 : 2;
  int64_t total = 0, tiles = 0;
  for (const Unit& u : units) {
    total += static_cast<int64_t>(u.tiles() + extra) * u.weight;
    tiles += std::max(1, u.tiles());
  }
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>(ctas, tiles));
  *slots = 0;
  *most = 1;
  if (place_whole(units, ctas, extra, group, window, items, first)) return;
  if (section == 0 && (flags & D2SD_PLAN_CLUSTERS) &&
      place_clusters(units, ctas, group, window, (flags & D2SD_PLAN_EIGHT_BIT) != 0, items, first, most))
    return;
  first.assign(1, 0);
  int64_t done = 0;  // cost handed out so far
  int32_t count = 0;
  for (const Unit& u : units) {
    const size_t at = items.size();
    const int64_t fixed = static_cast<int64_t>(extra) * u.weight;
    int32_t key = u.key0, parts = 0;
    int64_t left = u.tiles();
    do {
      // this CTA's share ends at cost total * k / n
      const int64_t k = static_cast<int64_t>(first.size());
      int64_t take = left;
      if (k < n) {
        const int64_t room = (total * k / n - done - fixed) / u.weight;
        take = std::min(left, std::max<int64_t>(room, 1));
        if (left - take == 1 && take > 1) take = left;  // no splinter of one tile
      }
      const int32_t end = take == left ? u.key1 : key + static_cast<int32_t>(take) * kTileKeys;
      const int32_t it[kItemInts] = {u.req,  u.head,     u.tok0,   u.row0, u.nrows, key, end, u.pos0,
                                     window, u.page_off, u.kv_len, parts,  0,       u.row0 / group, 0, 0};
      items.insert(items.end(), it, it + kItemInts);
      ++count;
      ++parts;
      left -= take;
      done += take * u.weight + fixed;
      if (left > 0) total += fixed;  // the next part's own
      key = end;
      // the next item starts in the CTA whose share still has room for a tile
      while (static_cast<int64_t>(first.size()) < n &&
             done + fixed + u.weight > total * static_cast<int64_t>(first.size()) / n)
        first.push_back(count);
    } while (left > 0);
    for (int p = 0; p < parts; ++p) {
      int32_t* it = items.data() + at + static_cast<size_t>(p) * kItemInts;
      it[P_SLOT] = parts > 1 ? *slots + p : -1;
      it[P_PARTS] = parts;
    }
    if (parts == 1) continue;
    for (int r = 0; r < u.nrows;) {  // rows of one q tile at a time
      const int tile = r / q_tile, in_tile = r % q_tile;
      const int n = std::min({kJoinRows[section], u.nrows - r, q_tile - in_tile});
      const int32_t j[kJoinInts] = {*slots * per + tile, per, parts, in_tile, n, u.row0 + r, u.tok0, u.head};
      joins.insert(joins.end(), j, j + kJoinInts);
      r += n;
    }
    *slots += parts;
    *most = std::max(*most, parts);
  }
  first.push_back(count);
}

}  // namespace
}  // namespace d2sd

extern "C" int64_t d2sd_paged_plan_capacity(const int32_t* q_lens, int32_t num_requests,
                                            int32_t num_qo_heads, int32_t num_kv_heads,
                                            int32_t num_ctas) {
  using namespace d2sd::paged;
  if (!q_lens || num_requests < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 ||
      num_qo_heads % num_kv_heads || num_ctas <= 0)
    return -1;
  const int64_t G = num_qo_heads / num_kv_heads;
  int64_t units = 0;
  for (int r = 0; r < num_requests; ++r) {
    if (q_lens[r] < 0) return -1;
    units += (q_lens[r] * G + kRowsTile - 1) / kRowsTile * num_kv_heads;
  }
  // every CTA adds at most one cut; a cut unit has at most 256 rows to join
  const int64_t ctas = section_ctas(0, num_ctas) + section_ctas(1, num_ctas);
  return kHeaderInts + (units + 2 * ctas) * kItemInts + 2 * (ctas + 8) +
         (static_cast<int64_t>(section_ctas(0, num_ctas)) * (kRowsTile / kJoinRows[0]) +
          static_cast<int64_t>(num_ctas) * (256 / kJoinRows[1])) * kJoinInts;
}

extern "C" int d2sd_paged_plan(const int32_t* q_lens, const int32_t* kv_lens,
                               const int32_t* page_offsets, int32_t num_requests, int32_t num_qo_heads,
                               int32_t num_kv_heads, int32_t causal, int32_t window, int32_t flags,
                               int32_t num_ctas, int32_t* plan, int64_t capacity, int64_t* used, int32_t* sections) {
  using namespace d2sd;
  using namespace d2sd::paged;
  if (num_requests < 0 || (num_requests > 0 && (!q_lens || !kv_lens || !page_offsets)) || !plan ||
      !used || !sections || num_ctas <= 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || window < 0)
    return plan_fail(D2SD_ERR_INVALID_ARGUMENT, "invalid argument");
  if (num_qo_heads % num_kv_heads)
    return plan_fail(D2SD_ERR_INVALID_ARGUMENT, "query heads must be a multiple of kv heads");
  if (window > 0 && !causal)
    return plan_fail(D2SD_ERR_UNSUPPORTED, "a window needs a causal mask");
  window = std::min(window, kNoLimit);  // positions are below it
  const int G = num_qo_heads / num_kv_heads;
  try {
    if (G > 128) return plan_fail(D2SD_ERR_UNSUPPORTED, "more than 128 query heads per kv head");
    std::vector<Unit> units[kSections];
    int64_t tok = 0;
    for (int r = 0; r < num_requests; ++r) {
      const int64_t n = q_lens[r], kv = kv_lens[r];
      if (n < 0 || kv < 0 || page_offsets[r] < 0)
        return plan_fail(D2SD_ERR_INVALID_ARGUMENT, "negative length or page offset");
      if (kv >= kNoLimit || n * G >= kNoLimit || tok + n >= kNoLimit)
        return plan_fail(D2SD_ERR_UNSUPPORTED, "lengths above 2^30");
      const int64_t rows = n * G;
      // few rows: tiles of 16 rows; else pairs of q tiles of whole tokens, where a
      // unit of one q tile works on two key tiles at a time
      const int section = rows <= (flags & D2SD_PLAN_EIGHT_BIT ? kRowsLimit8 : kRowsLimit) ? 0 : 1;
      const int64_t q_tile = static_cast<int64_t>(128 / G) * G;
      const int64_t tile = section == 0 ? kRowsTile : 2 * q_tile;
      const int32_t pos0 = causal ? static_cast<int32_t>(kv - n) : kNoLimit;
      for (int h = 0; h < num_kv_heads; ++h) {
        for (int64_t row = 0; row < rows; row += tile) {
          const int64_t nr = std::min(tile, rows - row);
          const int64_t t0 = row / G, t1 = (row + nr - 1) / G;
          int64_t lo = 0, hi = kv;
          if (causal) {
            hi = std::max<int64_t>(0, std::min<int64_t>(kv, pos0 + t1 + 1));
            if (window) lo = std::max<int64_t>(0, pos0 + t0 + 1 - window);
          }
          lo = lo / 16 * 16;  // whole pages
          if (lo > hi) lo = hi;
          units[section].push_back({r, h, static_cast<int32_t>(tok), static_cast<int32_t>(row),
                                    static_cast<int32_t>(nr), static_cast<int32_t>(lo),
                                    static_cast<int32_t>(hi), pos0, page_offsets[r],
                                    static_cast<int32_t>(kv),
                                    section == 1 && nr > q_tile ? 2 : 1});
        }
      }
      tok += n;
    }
    std::vector<int32_t> out(kHeaderInts, 0);
    out[H_MAGIC] = kMagic;
    out[H_REQUESTS] = num_requests;
    out[H_TOKENS] = static_cast<int32_t>(tok);
    out[H_GROUP] = G;
    out[H_KV_HEADS] = num_kv_heads;
    for (int s = 0; s < kSections; ++s) {
      int32_t sec[kSectionInts] = {0};
      if (!units[s].empty()) {
        std::vector<int32_t> items, first, joins;
        cut(units[s], section_ctas(s, num_ctas), s, G, window, flags, items, first, joins, &sec[S_SLOTS], &sec[S_PARTS]);
        sec[S_CTAS] = static_cast<int32_t>(first.size()) - 1;
        sec[S_ITEMS] = static_cast<int32_t>(items.size() / kItemInts);
        sec[S_OFF_CTA] = static_cast<int32_t>(out.size());
        out.insert(out.end(), first.begin(), first.end());
        while (out.size() % 4) out.push_back(0);
        sec[S_OFF_ITEMS] = static_cast<int32_t>(out.size());
        out.insert(out.end(), items.begin(), items.end());
        sec[S_JOINS] = static_cast<int32_t>(joins.size() / kJoinInts);
        sec[S_OFF_JOINS] = static_cast<int32_t>(out.size());
        out.insert(out.end(), joins.begin(), joins.end());
      }
      memcpy(out.data() + H_SECTION + s * kSectionInts, sec, sizeof(sec));
      memcpy(sections + s * kSectionInts, sec, sizeof(sec));
    }
    // the page-table entries that the tiles kernel's requests span, and how often its
    // units go over them
    int64_t visits = 0, lo = kNoLimit, hi = 0;
    for (const Unit& u : units[1]) {
      visits += static_cast<int64_t>(u.tiles()) * (kTileKeys / 16);
      lo = std::min<int64_t>(lo, u.page_off);
      hi = std::max<int64_t>(hi, u.page_off + static_cast<int64_t>(u.kv_len + 15) / 16);
    }
    int32_t* host = sections + kSections * kSectionInts;
    host[0] = host[1] = host[2] = host[3] = 0;
    for (const Unit& u : units[1]) host[3] |= u.weight > 1 ? 1 : 0;  // a unit of two q tiles
    for (const Unit& u : units[0]) host[3] |= u.nrows > 8 ? 2 : 0;   // of more than 8 rows
    if (hi > lo && hi < kNoLimit) {
      host[0] = static_cast<int32_t>(std::min<int64_t>(visits / ((hi - lo) * num_kv_heads), kNoLimit));
      host[1] = static_cast<int32_t>(lo);
      host[2] = static_cast<int32_t>(hi);
    }
    *used = static_cast<int64_t>(out.size());
    if (*used > capacity) return plan_fail(D2SD_ERR_WORKSPACE, "plan buffer too small");
    memcpy(plan, out.data(), out.size() * sizeof(int32_t));
  } catch (const std::exception& e) {  // out of host memory
    return plan_fail(D2SD_ERR_INVALID_ARGUMENT, e.what());
  }
  return D2SD_OK;
}
