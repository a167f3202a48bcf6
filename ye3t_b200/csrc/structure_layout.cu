// Work tables of a batch for structure attention, built on the host (the layout in include/ye3t_b200.h).
//
// Which kernel computes which structure:
//   small   up to 64 queries and 64 keys, where all structures are small or the small ones fill the SMs by
//           themselves (a tile of 128 rows would be mostly empty, but a launch for a few structures costs more than it
//           saves: 4 molecules beside 12 clusters of some hundred atoms, 362 us against 201 in a training step);
//   row     no or a single key: its weight is exactly 1 and its gradients through the softmax exactly 0, which the
//           row kernels keep;
//   few     up to two queries: a tile would hold 2 rows of 128 (8 structures of 16,384 keys, 8 heads: 111 us on tiles,
//           64 on the few-query kernels; their keys' gradients 209 us on tiles, 111 by a few lanes a key, in items of 128
//           keys: with an entry a key the tables of 8 structures of 14,000 keys took 701 us and 889 KB on the host, in
//           items 22 us and 33 KB);
//   tile    the rest.
// A tile's columns are cut into parts, which are joined, where that makes the last wave of CTAs shorter (16,384 atoms, 8
// heads: forward 1,273 us and 39 to join against 1,431 uncut, when P had one piece).
#include <algorithm>
#include <iterator>
#include <new>
#include <vector>

#include "common.cuh"

namespace y3b {
namespace {

constexpr int64_t kTile = 128, kSmall = 64, kFew = 2;

struct Side {
  std::vector<int32_t> items, joins, rows;
  int64_t slots = 0;
};

struct Range {
  int64_t first, count;
};

struct Part {
  int32_t row, rows, col, cols, slot;
};

// How many parts a tile of `cols` columns is cut into: all alike, or only those past the last full wave.  CTAs cost
// kStart columns of time to start and finish, and a part kJoin more to be joined.
constexpr int64_t kStart = 96, kJoin = 64, kMostParts = 8;

struct Cut {
  int64_t all = 1, last = 1, from = 0;  // tiles from number `from` on are cut into `last` parts, those before into `all`
};

// Tiles of equal length on `slots` places for a tile (over all heads): the cheapest number of waves.
Cut cut_evenly(int64_t tiles, int64_t cols, int64_t slots) {
  Cut best;
  best.from = tiles;
  const auto waves = [&](int64_t n) { return (n + slots - 1) / slots; };
  int64_t least = waves(tiles) * (cols + kStart);
  for (int64_t n = 2; n <= kMostParts && cols / n >= 256; ++n) {
    const int64_t part = cols / n + kStart + kJoin;
    if (waves(tiles * n) * part < least) {
      least = waves(tiles * n) * part;
      best.all = best.last = n;
      best.from = tiles;
    }
    const int64_t full = tiles / slots * slots;
    const int64_t cost = full / slots * (cols + kStart) + waves((tiles - full) * n) * part;
    if (full > 0 && cost < least) {
      least = cost;
      best.all = 1;
      best.last = n;
      best.from = full;
    }
  }
  return best;
}

// Tiles of the structures in `which`: rows [row] and columns [col] of each, on `slots` places over all heads; `always`
// joins every tile.
void add_tiles(Side* side, const std::vector<Range>& row, const std::vector<Range>& col,
               const std::vector<int64_t>& which, int64_t heads, int64_t slots, bool always) {
  int64_t work = 0, tiles = 0;
  bool even = !which.empty() && !always;
  for (const int64_t s : which) {
    const int64_t n = (row[s].count + kTile - 1) / kTile;
    tiles += n;
    work += n * std::max<int64_t>(col[s].count, 1);
    even = even && col[s].count == col[which[0]].count;
  }
  // parts of tiles of many lengths: no longer than what a place would get of the whole
  const int64_t chunk = std::max<int64_t>(always ? 128 : 256, work * heads / slots);
  const Cut cut = even ? cut_evenly(tiles * heads, col[which[0]].count, slots) : Cut{};
  std::vector<Part> parts;
  int64_t tile = 0;
  for (const int64_t s : which) {
    for (int64_t r = 0; r < row[s].count; r += kTile, ++tile) {
      const int64_t n = even ? (tile * heads >= cut.from ? cut.last : cut.all)
                             : std::max<int64_t>(1, (2 * col[s].count + chunk) / (2 * chunk));
      const int64_t step = ((col[s].count + n - 1) / n + 63) / 64 * 64;  // parts begin at multiples of 64 columns
      const int32_t first = int32_t(row[s].first + r), rows = int32_t(std::min(kTile, row[s].count - r));
      const bool split = n > 1 || always;
      if (split) {
        const int32_t join[4] = {first, rows, int32_t(side->slots), int32_t(n)};
        side->joins.insert(side->joins.end(), join, join + 4);
      }
      for (int64_t k = 0; k < n; ++k) {
        const int64_t b = std::min(k * step, col[s].count), e = std::min(b + step, col[s].count);
        parts.push_back({first, rows, int32_t(col[s].first + b), int32_t(e - b),
                         split ? int32_t(side->slots + k) : -1});
      }
      if (split) side->slots += n;
    }
  }
  // the longest first: the last CTAs to start are short
  std::stable_sort(parts.begin(), parts.end(), [](const Part& a, const Part& b) { return a.cols > b.cols; });
  side->items.reserve(parts.size() * 8);
  for (const Part& p : parts) {
    const int32_t item[8] = {p.row, p.rows, p.col, p.cols, p.slot, 0, 0, 0};
    side->items.insert(side->items.end(), item, item + 8);
  }
}

void add_rows(Side* side, const std::vector<Range>& row, const std::vector<int64_t>& which) {
  for (const int64_t s : which) {
    for (int64_t r = 0; r < row[s].count; ++r) {
      side->rows.push_back(int32_t(row[s].first + r));
      side->rows.push_back(int32_t(s));
    }
  }
}

// Keys whose structure has one or two queries, in items of up to kTile of one structure.
void add_few_keys(Side* side, const std::vector<Range>& key, const std::vector<Range>& query,
                  const std::vector<int64_t>& which) {
  for (const int64_t s : which) {
    for (int64_t r = 0; r < key[s].count; r += kTile) {
      const int32_t item[8] = {int32_t(key[s].first + r), int32_t(std::min(kTile, key[s].count - r)),
                               int32_t(query[s].first), int32_t(query[s].count), -1, 0, 0, 0};
      side->items.insert(side->items.end(), item, item + 8);
    }
  }
}

int64_t build(const int64_t* queries, const int64_t* keys, int64_t n, int64_t heads, int64_t key_heads,
              int64_t* counts, int32_t* out, int64_t capacity) {
  std::vector<Range> q(n), k(n);
  int64_t nq = 0, nk = 0;
  for (int64_t s = 0; s < n; ++s) {
    q[s] = {nq, queries[s]};
    k[s] = {nk, keys[s]};
    nq += queries[s];
    nk += keys[s];
  }
  int64_t small_count = 0;
  for (int64_t s = 0; s < n; ++s) small_count += queries[s] <= kSmall && keys[s] <= kSmall;
  const bool use_small = small_count == n || small_count * key_heads >= 2 * kSMs;
  std::vector<int64_t> low, high, by_row, few, tiled, key_tiled;
  for (int64_t s = 0; s < n; ++s) {
    if (use_small && queries[s] <= kSmall && keys[s] <= kSmall) {
      if (queries[s] > kSmall / 2 || keys[s] > kSmall / 2) high.push_back(s);
      else if (queries[s] + keys[s] > 0) low.push_back(s);
    } else if (keys[s] <= 1) {
      by_row.push_back(s);
    } else {
      if (queries[s] > kFew) tiled.push_back(s);
      else if (queries[s] > 0) few.push_back(s);
      if (queries[s] > kFew || queries[s] == 0) key_tiled.push_back(s);
    }
  }
  // Places: two CTAs an SM of the tile kernels; four of the few-query kernels.  The forward's are counted as those of the
  // kernel that takes two heads a CTA, where their number is even: a layout knows neither the type nor the width, and
  // that kernel (bf16 with distances, widths up to 64) gains more by it (8,192 atoms, 8 heads of 64: 410 us against 454 cut
  // for half the places; 16,384 atoms 1,423 and 1,414) than the others mostly lose (fp32, 4,096 atoms, 4 heads of 64: 164 us
  // against 158; 8,192 atoms 535 and 534; 16 clusters of 300, 8 heads on 2, fp32: 70 and 58; bf16, 8,192 atoms, 8 heads of
  // 128: 565 and 538).
  Side forward, query, key, one;
  add_tiles(&forward, q, k, tiled, heads, kSMs * (heads % 2 == 0 ? 4 : 2), false);
  add_tiles(&query, q, k, tiled, heads, kSMs * 2, false);
  add_tiles(&key, k, q, key_tiled, key_heads, kSMs * 2, false);
  add_tiles(&one, q, k, few, key_heads, kSMs * 4, true);
  add_rows(&query, q, by_row);
  add_rows(&key, k, by_row);
  const int64_t key_tiles = int64_t(key.items.size()) / 8;
  add_few_keys(&key, k, q, few);
  const auto entries = [](const std::vector<int32_t>& v, int width) { return int64_t(v.size()) / width; };
  const int64_t all[] = {int64_t(low.size()),      int64_t(high.size()),     entries(one.items, 8),
                         entries(one.joins, 4),    entries(forward.items, 8), entries(forward.joins, 4),
                         forward.slots,            entries(query.items, 8),  entries(query.joins, 4),
                         query.slots,              entries(query.rows, 2),   entries(key.items, 8),
                         entries(key.joins, 4),    key.slots,                entries(key.rows, 2),
                         entries(key.items, 8) - key_tiles};
  static_assert(sizeof(all) == 16 * sizeof(int64_t), "what callers reserve for counts");
  std::copy(std::begin(all), std::end(all), counts);
  const std::vector<int32_t>* const tables[] = {&forward.items, &query.items, &key.items, &one.items,
                                                &forward.joins, &query.joins, &key.joins, &one.joins};
  int64_t need = 4 * int64_t(low.size() + high.size()) + int64_t(query.rows.size() + key.rows.size()) + 2 * (n + 1);
  for (const auto* t : tables) need += int64_t(t->size());
  if (!out || capacity < need) return need;
  for (const auto* t : tables) out = std::copy(t->begin(), t->end(), out);
  for (const auto* list : {&low, &high}) {
    for (const int64_t s : *list) {
      const int64_t entry[4] = {q[s].first, q[s].count, k[s].first, k[s].count};
      for (const int64_t v : entry) *out++ = int32_t(v);
    }
  }
  out = std::copy(query.rows.begin(), query.rows.end(), out);
  out = std::copy(key.rows.begin(), key.rows.end(), out);
  for (int64_t s = 0; s < n; ++s) *out++ = int32_t(q[s].first);
  *out++ = int32_t(nq);
  for (int64_t s = 0; s < n; ++s) *out++ = int32_t(k[s].first);
  *out++ = int32_t(nk);
  return need;
}

}  // namespace
}  // namespace y3b

using namespace y3b;

extern "C" int64_t y3b_structure_layout(const int64_t* query_counts, const int64_t* key_counts, int64_t structure_count,
                                        int64_t heads, int64_t key_heads, int64_t* counts, int32_t* tables,
                                        int64_t capacity) {
  Y3B_CHECK_ARG(structure_count >= 0 && structure_count < INT32_MAX, "structure_layout: bad structure count");
  Y3B_CHECK_ARG(counts && (structure_count == 0 || (query_counts && key_counts)), "structure_layout: null argument");
  Y3B_CHECK_ARG(heads >= 1 && key_heads >= 1 && heads % key_heads == 0 && heads <= 1024,
                "structure_layout: the query heads must be a multiple of the key heads, 1024 at most");
  int64_t nq = 0, nk = 0;
  for (int64_t s = 0; s < structure_count; ++s) {
    Y3B_CHECK_ARG(query_counts[s] >= 0 && key_counts[s] >= 0, "structure_layout: negative count");
    Y3B_CHECK_ARG(query_counts[s] <= INT32_MAX - nq && key_counts[s] <= INT32_MAX - nk,
                  "structure_layout: at most 2^31 - 1 atoms in a batch");
    nq += query_counts[s];
    nk += key_counts[s];
  }
  try {
    return build(query_counts, key_counts, structure_count, heads, key_heads, counts, tables, capacity);
  } catch (const std::bad_alloc&) {
    return fail(Y3B_ERR_ARGUMENT, "structure_layout: out of host memory");
  }
}
