// Work lists of the unmasked attention forms (segment_attn.cu): attention to an encoder's states, and attention
// of a batch that shares a long prefix.  Host code only.
//
// Both are made of two kinds of work:
//   tiles   up to 256 (token, query head) rows of one kv head, or up to 128 of each of two, against one range of keys that all of them see, on
//           the tensor cores (the tokens of a sequence against its encoder's states; all the tokens of a batch
//           against the shared prefix);
//   items   one token against a range of its own keys, on the decode kernels (sequences with few tokens; each
//           token's keys behind the prefix).
// A token that is worked on in one piece is written by the kernel that does it; of any other every piece leaves a
// partial (maximum, sum, accumulator), and the merge kernel folds them.
//
// Tiles are dealt to blocks here, one list of items for each block of the tile kernel (one per SM): either whole, the
// longest first to the block with the least to do, or laid end to end and cut into equal shares, whichever ends first.
//
// The launches of a step are made for its counts and offsets, so each of them looks at the image's stamp, which names these, first.
//
// Image in the workspace (every region 256-byte aligned, offsets in pkv_segment_plan):
//   PlanHeader | token_seq[n_tokens] | token_pos[n_tokens] | row_token[..] | WorkItem[..] (and the first item of every
//   share) | int first tile of every list, and the end | TileItem[..] | MergeRow[..]
// and behind it the partials.  Of the tiles: float2 (maximum, sum) [row], float [row][head_dim], where an item's rows lie
// one behind the other; of the decode kernels: float2 [part][q_heads], float [part][q_heads][head_dim].
#pragma once
#include <algorithm>
#include <cstring>
#include <functional>
#include <map>
#include <queue>
#include <utility>
#include <vector>

#include "decode_list.hpp"
#include "decode_plan.hpp"
#include "status.hpp"

namespace pkv {

constexpr int kTileRows = 256;      // rows of a tile item: two groups of 128
constexpr int kTileKeys = 128;      // keys per step of the tile kernel
// What its waits for whole items allow (2.1 s): keys of an item, walked in 0.6 s, and a block's list, in cycles (1.1 s).
constexpr int kMostTileKeys = 1 << 25;
constexpr long long kMostListCycles = 2000000000ll;

// Tokens row_token[tok0 .. tok0 + n_tok - 1] of a segment: row r of the item is token r / group, head r % group.
struct TileItem {
  int tok0, n_tok, kvh;
  int kv_begin, kv_len;             // kv_begin a multiple of kTileKeys
  int part;                         // first of its partial rows, or -1: write the output
  int flags;
  int source;                       // whose block table: the sequence of this token, or (< 0) sequence ~source
};
constexpr int kConsecutive = 1;     // the tokens are consecutive rows of q
constexpr int kPair = 2;            // at most 128 rows, of kv head kvh for one group and kvh + 1 for the other
// Partials of a token's heads of one kv head: of tiles, n_tile of them, tile_stride rows apart; of the decode kernels, n_own.
// None at all: there are no keys, the output is zero.
struct MergeRow { int token, kvh, tile_row, tile_stride, n_tile, own_part, n_own, pad; };

struct SegmentGeometry {
  int n_tokens, q_heads, kv_heads, head_dim, block_size, elem_bytes;
  int group() const { return q_heads / kv_heads; }
  int tile_tokens() const { return kTileRows / group(); }      // of a full tile
  // whether the tile kernel is written for it
  bool tiles() const {
    return elem_bytes == 2 && group() <= kTileRows && (head_dim == 64 || head_dim == 128) && block_size >= 16 && (block_size & (block_size - 1)) == 0;
  }
};

// A sequence whose tokens (row_token[tok0 .. tok0 + n_tok - 1]) all see keys 0 .. kv_len - 1.
struct Segment { int tok0, n_tok, kv_len, source; };   // source: as in its tiles
// A token of the decode kernels: keys begin .. begin + len - 1, len > 0.
struct OwnRange { int token, begin, len; };

struct SegmentLists {
  std::vector<int> row_token;
  std::vector<WorkItem> items;
  std::vector<int> first;           // of every share, and the end; empty: no shares
  std::vector<int> list_first;      // tiles of every block
  std::vector<TileItem> tiles;
  std::vector<MergeRow> merge;
  long long n_tile_rows = 0;
  long long list_cycles = 0;        // of the longest list
  int n_parts = 0, chunk = 0, longest = 0;
};

inline int own_extra(const SegmentGeometry& g) { return decode_max_extra(g.kv_heads); }
// Most partials of a step.  A block's list begins and ends with a piece of a tile at most; prefix steps leave one of
// each kind per token even where nothing is cut.
inline long long most_tile_rows(const SegmentGeometry& g, int sms, bool prefix) {
  return 2ll * sms * kTileRows + (prefix ? static_cast<long long>(g.n_tokens) * g.q_heads : 0ll);
}
inline long long most_parts(const SegmentGeometry& g, bool prefix) { return (prefix ? g.n_tokens : 0ll) + 2ll * own_extra(g); }

// What the planner reckons with, in cycles of 1/1.75 ns (measured on B200; head_dim 64 and 128 alike within a tenth).
// A block of the tile kernel: an item's start and end, and a key tile of two groups, of one alone, of a pair of heads.
constexpr int kItemCycles = 5000, kTwoGroupCycles = 3700, kOneGroupCycles = 3500, kPairCycles = 4200;
constexpr int kLeastTiles = 2;      // key tiles of a piece, at least
constexpr int kManyUnits = 32;      // units a block, from which on a step's time is their average
constexpr int kFewUnits = 2;        // and up to which it is worth while to look for fewer blocks
// Partials of tiles are written and read at about 2,000 bytes a cycle, and the merge is a launch more.
constexpr int kMergeCycles = 5000;
inline long long partial_cycles(long long rows, int head_dim) { return rows * head_dim * 8 / 2000; }
// The decode kernels: a launch, and the K/V of every token's keys, mostly from L2.  (64 tokens of 1,084 keys on 8 kv heads of
// 128 dims 31 us by this account and measured; 6 of 560 on 2 of 64 4.7 and 3.7.)
constexpr int kOwnCycles = 7900, kOwnBytesPerCycle = 6300;
inline long long own_fetch(const std::vector<OwnRange>& own, const SegmentGeometry& g) {
  long long keys = 0;
  for (const OwnRange& o : own) keys += o.len;
  return keys * g.kv_heads * g.head_dim * 2 * g.elem_bytes / kOwnBytesPerCycle;
}
inline long long own_cycles(const std::vector<OwnRange>& own, const SegmentGeometry& g) { return own.empty() ? 0 : kOwnCycles + own_fetch(own, g); }
// Behind a tile kernel: their blocks start on the SMs that it leaves free, kOwnStart cycles after it, and what is left when it ends takes
// the whole GPU and kOwnTail more.  (128 tokens behind 2,048 keys, 32/4 heads of 64: 128 blocks of tiles 20.6 us, 64 blocks of
// twice as many 15.9.  200 behind 16,384, 32/8 of 128: 148 blocks 87.3 us, 132 84.8, 139 84.0, 112 85.4, 96 95.4.)
constexpr int kOwnStart = 6000, kOwnTail = 4000;

struct TileUnit { TileItem item; int n_kt, per_tile; long long cycles() const { return kItemCycles + static_cast<long long>(n_kt) * per_tile; } };
struct TileDeal {
  std::vector<std::vector<TileItem>> lists;
  int blocks = 0;                                                          // lists
  long long cycles = 0, part_rows = 0, cost = 0;                           // of the longest list; with the partials' way
};
// With the decode kernels' part behind it, `fetch` cycles on the whole GPU.
inline long long joint_cost(const TileDeal& d, long long fetch, int sms) {
  const long long hidden = std::max<long long>(d.cycles - kOwnStart, 0) * (sms - d.blocks) / sms;
  return d.cost + (fetch > hidden ? fetch - hidden + kOwnTail : 0);
}

inline long long item_rows(const TileItem& t, const SegmentGeometry& g) { return static_cast<long long>(t.n_tok) * g.group() * (t.flags & kPair ? 2 : 1); }

// Whole, longest first, each to the block with the least to do so far.  `keep`: the lists, not only what they would cost.
inline TileDeal deal_whole(const std::vector<TileUnit>& units, int sms, bool keep) {
  std::vector<int> order(units.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = static_cast<int>(i);
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return units[x].cycles() > units[y].cycles(); });
  TileDeal d;
  const size_t blocks = std::min<size_t>(units.size(), sms);
  d.blocks = static_cast<int>(blocks);
  if (keep) d.lists.resize(blocks);
  using Load = std::pair<long long, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least;
  for (size_t b = 0; b < blocks; ++b) least.push({0, static_cast<int>(b)});
  for (int u : order) {
    Load l = least.top();
    least.pop();
    if (keep) d.lists[l.second].push_back(units[u].item);
    l.first += units[u].cycles();
    d.cycles = std::max(d.cycles, l.first);
    least.push(l);
  }
  d.cost = d.cycles;
  return d;
}

// End to end, cut into equal shares.  `part` numbers the pieces' partial rows; pieces of a unit lie one behind the other.
inline TileDeal deal_shares(const std::vector<TileUnit>& units, int sms, int least, const SegmentGeometry& g, bool prefix, bool keep) {
  TileDeal d;
  long long total = 0, longest = 0;
  for (const TileUnit& u : units) {
    total += u.cycles();
    longest = std::max<long long>(longest, u.per_tile);
  }
  // every cut costs an item's start and end again
  const long long share = std::max<long long>((total + static_cast<long long>(sms) * kItemCycles) / sms, kItemCycles + least * longest);
  long long room = 0, done = 0;
  int lists = 0, in_list = 0;                                              // so far; items of the last one
  std::vector<std::pair<size_t, size_t>> pieces;                           // of a unit: (list, place)
  for (const TileUnit& u : units) {
    int n_pieces = 0;
    pieces.clear();
    for (int at = 0; at < u.n_kt;) {
      const bool last = lists >= sms;
      if (lists == 0 || (!last && in_list > 0 && room < kItemCycles + std::min(kLeastTiles, u.n_kt - at) * static_cast<long long>(u.per_tile))) {
        ++lists;
        if (keep) d.lists.emplace_back();
        room += share;                                                     // (what a list leaves, the next one gets)
        done = in_list = 0;
        continue;
      }
      int n = last ? u.n_kt - at : static_cast<int>(std::min<long long>(u.n_kt - at, std::max<long long>(kLeastTiles, (room - kItemCycles) / u.per_tile)));
      if (u.n_kt - at - n < kLeastTiles) n = u.n_kt - at;                  // nothing worth a piece would be left
      if (keep) {
        TileItem t = u.item;
        t.kv_begin = at * kTileKeys;
        t.kv_len = std::min(n * kTileKeys, u.item.kv_len - t.kv_begin);
        pieces.push_back({d.lists.size() - 1, d.lists.back().size()});
        d.lists.back().push_back(t);
      }
      ++n_pieces;
      ++in_list;
      const long long took = kItemCycles + static_cast<long long>(n) * u.per_tile;
      room -= took;
      done += took;
      d.cycles = std::max(d.cycles, done);
      at += n;
    }
    if (prefix || n_pieces > 1) {
      const long long rows = item_rows(u.item, g);
      for (size_t p = 0; p < pieces.size(); ++p) d.lists[pieces[p].first][pieces[p].second].part = static_cast<int>(d.part_rows + static_cast<long long>(p) * rows);
      d.part_rows += n_pieces * rows;
    }
  }
  d.blocks = lists;
  d.cost = d.cycles + (d.part_rows > 0 ? (prefix ? 0 : kMergeCycles) + partial_cycles(d.part_rows, g.head_dim) : 0);
  return d;
}

// Cuts the decode kernels' tokens, as pkv_decode_plan_host does: equal shares where there are enough keys, else chunks,
// longest first.  pieces[i]: how many the i-th has; the items' `part` is the piece's number until it is known where
// the token's partials begin.
inline void cut_own(const std::vector<OwnRange>& own, const SegmentGeometry& g, int extra, SegmentLists& out, std::vector<int>& pieces) {
  long long total = 0;
  out.longest = 0;
  for (const OwnRange& o : own) {
    total += share_padded(o.len);
    out.longest = std::max(out.longest, o.len);
  }
  pieces.assign(own.size(), 1);
  if (own.empty()) return;
  const ShareRule rule = share_rule(total, out.longest, static_cast<int>(own.size()),
                                    decode_plan_limits(extra, g.q_heads, g.kv_heads, g.head_dim), false);
  out.chunk = rule.per > 0 ? rule.per : rule.chunk;
  if (rule.per > 0) {
    long long begin = 0;
    for (size_t i = 0; i < own.size(); ++i) {
      const OwnRange& o = own[i];
      const ShareCut cut = share_cuts(begin, share_padded(o.len), rule.per);
      pieces[i] = cut.n + 1;
      for (int s = 0; s <= cut.n; ++s) {
        const long long at = s ? cut.first + static_cast<long long>(s - 1) * rule.per : begin;
        const int b = static_cast<int>(at - begin);
        const int e = s < cut.n ? static_cast<int>(cut.first + static_cast<long long>(s) * rule.per - begin) : o.len;
        for (const int sh = share_of(at, rule.per, rule.n_shares); static_cast<int>(out.first.size()) <= sh;)
          out.first.push_back(static_cast<int>(out.items.size()));
        out.items.push_back(WorkItem{static_cast<int>(i), o.begin + b, e - b, s});
      }
      begin += share_padded(o.len);
    }
    while (static_cast<int>(out.first.size()) <= rule.n_shares) out.first.push_back(static_cast<int>(out.items.size()));
    return;
  }
  const int chunk = rule.chunk > 0 ? rule.chunk : 0x40000000;
  for (size_t i = 0; i < own.size(); ++i) {
    pieces[i] = (own[i].len + chunk - 1) / chunk;
    for (int s = 0; s < pieces[i]; ++s)
      out.items.push_back(WorkItem{static_cast<int>(i), own[i].begin + s * chunk, std::min(chunk, own[i].len - s * chunk), s});
  }
  std::stable_sort(out.items.begin(), out.items.end(), [](const WorkItem& x, const WorkItem& y) { return x.kv_len > y.kv_len; });
}

// The cheapest of: whole, and shares of pieces of at least 2, 4, 8 ... key tiles (fewer pieces leave fewer partials), and with work
// for the decode kernels (`fetch`) each of them on fewer blocks too.
inline TileDeal deal_tiles(const std::vector<TileUnit>& units, long long fetch, int sms, const SegmentGeometry& g, bool prefix, bool keep) {
  if (units.empty()) return TileDeal();
  int pick = 0, on = sms, longest = 0;                                     // least tiles of a piece, 0: whole; blocks
  long long total = 0;
  for (const TileUnit& u : units) {
    longest = std::max(longest, u.n_kt);
    total += u.cycles();
  }
  if (!keep && units.size() > static_cast<size_t>(kManyUnits) * sms) {     // dealt out as good as evenly, whatever the order
    TileDeal d;
    if (prefix)
      for (const TileUnit& u : units) d.part_rows += item_rows(u.item, g);
    d.blocks = sms;
    d.cycles = total / sms;
    d.cost = d.cycles + partial_cycles(d.part_rows, g.head_dim);
    return d;
  }
  const bool narrow = fetch > 0 && units.size() <= static_cast<size_t>(kFewUnits) * sms;
  long long best = -1;
  for (int blocks = sms; blocks >= sms / 4; blocks -= std::max(sms / 16, 1)) {
    if (best >= 0 && total / blocks >= best) break;
    auto offer = [&](const TileDeal& d, int least) {
      const long long c = joint_cost(d, fetch, sms);
      if (best < 0 || c < best) { best = c; pick = least; on = blocks; }
    };
    bool level = false;
    if (!prefix) {
      const TileDeal d = deal_whole(units, blocks, false);
      offer(d, 0);
      // Cuts could gain a fiftieth and their merge's cost at most: whole without reckoning them.  (Many units are level by themselves.)
      level = d.cost <= total / blocks + total / blocks / 50 + kMergeCycles;
    }
    for (int least = kLeastTiles; !level; least *= 2) {
      const TileDeal d = deal_shares(units, blocks, least, g, prefix, false);
      if (d.part_rows <= most_tile_rows(g, sms, prefix)) offer(d, least);
      if (least >= longest) break;
    }
    if (!narrow) break;
  }
  return pick ? deal_shares(units, on, pick, g, prefix, keep) : deal_whole(units, on, keep);
}

inline std::vector<TileUnit> tile_units(const std::vector<Segment>& segs, const SegmentGeometry& g, const std::vector<int>& row_token) {
  const int group = g.group();
  std::vector<TileUnit> units;
  for (const Segment& s : segs) {
    const int n_kt = (s.kv_len + kTileKeys - 1) / kTileKeys;
    for (int kvh = 0; kvh < g.kv_heads; ++kvh)
      for (int t = 0; t < s.n_tok; t += g.tile_tokens()) {
        const int n = std::min(g.tile_tokens(), s.n_tok - t), tok0 = s.tok0 + t;
        const bool small = n * group <= kTileRows / 2, pair = small && (kvh ^ 1) < g.kv_heads;
        if (pair && (kvh & 1)) continue;
        const bool row = row_token[tok0 + n - 1] - row_token[tok0] == n - 1;              // (they ascend)
        units.push_back(TileUnit{TileItem{tok0, n, kvh, 0, s.kv_len, -1, (row ? kConsecutive : 0) | (pair ? kPair : 0), s.source}, n_kt,
                                 pair ? kPairCycles : small ? kOneGroupCycles : kTwoGroupCycles});
      }
  }
  return units;
}

// What a step would take with these tiles and own ranges.
inline long long step_cycles(const std::vector<Segment>& segs, const std::vector<OwnRange>& own, const std::vector<int>& row_token, const SegmentGeometry& g,
                             int sms, bool prefix) {
  if (segs.empty()) return own_cycles(own, g);
  const long long fetch = own_fetch(own, g);
  return joint_cost(deal_tiles(tile_units(segs, g, row_token), fetch, sms, g, prefix, false), fetch, sms) + (prefix ? kMergeCycles : 0);
}

// Puts everything together.  out.row_token holds the segments' tokens already; `empty`: tokens without keys.
inline void list_segments(const std::vector<Segment>& segs, const std::vector<OwnRange>& own, const std::vector<int>& empty, const SegmentGeometry& g,
                          int sms, bool prefix, SegmentLists& out) {
  std::vector<int> pieces;
  cut_own(own, g, own_extra(g), out, pieces);
  const int group = g.group();
  const std::vector<TileUnit> units = tile_units(segs, g, out.row_token);
  if (!units.empty()) {
    const TileDeal deal = deal_tiles(units, own_fetch(own, g), sms, g, prefix, true);
    out.n_tile_rows = deal.part_rows;
    out.list_cycles = deal.cycles;
    for (const auto& list : deal.lists) {
      out.list_first.push_back(static_cast<int>(out.tiles.size()));
      out.tiles.insert(out.tiles.end(), list.begin(), list.end());
    }
    out.list_first.push_back(static_cast<int>(out.tiles.size()));
  }
  // what is merged: tokens of tiles with partials, one record for each kv head, found through the tile's first piece
  std::vector<int> own_of(g.n_tokens, -1), base(own.size(), -1);
  for (size_t i = 0; i < own.size(); ++i) own_of[own[i].token] = static_cast<int>(i);
  std::vector<char> seen(own.size(), 0);
  auto parts_of = [&](int o) {
    if (base[o] < 0) {
      base[o] = out.n_parts;
      out.n_parts += pieces[o];
    }
    return base[o];
  };
  std::map<std::pair<int, int>, int> n_pieces;                                            // of a unit: (tok0, kvh)
  for (const TileItem& t : out.tiles)
    if (t.part >= 0) ++n_pieces[{t.tok0, t.kvh}];
  for (const TileItem& t : out.tiles) {
    if (t.part < 0 || t.kv_begin > 0) continue;
    const int rows = t.n_tok * group, heads = t.flags & kPair ? 2 : 1, n = n_pieces[{t.tok0, t.kvh}];
    for (int h = 0; h < heads; ++h)
      for (int i = 0; i < t.n_tok; ++i) {
        const int token = out.row_token[t.tok0 + i], o = own_of[token];
        out.merge.push_back(MergeRow{token, t.kvh + h, t.part + h * rows + i * group, heads * rows, n, o >= 0 ? parts_of(o) : 0, o >= 0 ? pieces[o] : 0, 0});
        if (o >= 0) seen[o] = 1;
      }
  }
  for (size_t i = 0; i < own.size(); ++i)
    if (!seen[i] && pieces[i] > 1)
      for (int kvh = 0, at = parts_of(static_cast<int>(i)); kvh < g.kv_heads; ++kvh)
        out.merge.push_back(MergeRow{own[i].token, kvh, 0, 0, 0, at, pieces[i], 0});
  for (WorkItem& w : out.items) {
    const int i = w.token;
    w.token = own[i].token;
    w.part = base[i] < 0 ? -1 : base[i] + w.part;
  }
  for (int t : empty)
    for (int kvh = 0; kvh < g.kv_heads; ++kvh) out.merge.push_back(MergeRow{t, kvh, 0, 0, 0, 0, 0, 0});
}

}  // namespace pkv
