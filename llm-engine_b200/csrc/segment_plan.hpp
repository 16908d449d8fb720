// Work lists of the unmasked attention forms (segment_attn.cu): attention to an encoder's states, and attention
// of a batch that shares a long prefix.  Host code only.
//
// Both are made of two kinds of work:
//   tiles   up to 256 (token, query head) rows of one kv head against one range of keys that all of them see, on
//           the tensor cores (the tokens of a sequence against its encoder's states; all the tokens of a batch
//           against the shared prefix);
//   items   one token against a range of its own keys, on the decode kernels (sequences with few tokens; each
//           token's keys behind the prefix).
// A token that is worked on in one piece is written by the kernel that does it; of any other every piece leaves a
// partial (maximum, sum, accumulator), and the merge kernel folds them.
//
// Image in the workspace (every region 256-byte aligned, offsets in pkv_segment_plan):
//   PlanHeader | token_seq[n_tokens] | token_pos[n_tokens] | RowToken[..] | WorkItem[..] (and the first item of every
//   share) | TileItem[..] | MergeRow[..]
// and behind it the partials: float2 (maximum, sum) [part][q_heads], float [part][q_heads][head_dim].
#pragma once
#include <algorithm>
#include <cstring>
#include <vector>

#include "decode_list.hpp"
#include "decode_plan.hpp"
#include "status.hpp"

namespace pkv {

constexpr int kTileRows = 256;      // rows of a tile item: two groups of 128
constexpr int kTileKeys = 128;      // keys per step of the tile kernel

struct RowToken { int token, part_base; };
// The rows of tokens row_tokens[tok0 ..] of a segment: row r is token r / group, head r % group.
struct TileItem {
  int tok0, n_tok;
  int kv_begin, kv_len;             // kv_begin a multiple of kTileKeys
  int part;                         // partial slot behind the token's part_base, or -1: write the output
  int flags;
  int halves;                       // 1: at most 128 rows; the two groups take every other key tile, partials part and part + 1
  int pad;
};
constexpr int kConsecutive = 1;     // the tokens are consecutive rows of q
constexpr int kEmptySecond = 2;     // the others of the segment are halved: leave an empty partial part + 1
struct MergeRow { int token, part_base, n_parts, pad; };   // n_parts 0: no keys, the output is zero

struct SegmentGeometry {
  int n_tokens, q_heads, kv_heads, head_dim, block_size, elem_bytes;
  int group() const { return q_heads / kv_heads; }
  int tile_tokens() const { return kTileRows / group(); }      // of a full tile
  // whether the tile kernel is written for it
  bool tiles() const {
    return elem_bytes == 2 && group() <= kTileRows && (head_dim == 64 || head_dim == 128) && block_size >= 16 && (block_size & (block_size - 1)) == 0;
  }
};

// A sequence whose tokens (row_tokens[tok0 .. tok0 + n_tok - 1]) all see keys 0 .. kv_len - 1.
struct Segment {
  int tok0, n_tok, kv_len;
  int chunks, slots;                // ranges its keys are cut into; partials each of its tokens gets from them
};
// A token of the decode kernels: keys begin .. begin + len - 1, len > 0.
struct OwnRange { int token, begin, len; };

struct SegmentLists {
  std::vector<RowToken> rows;
  std::vector<WorkItem> items;
  std::vector<int> first;           // of every share, and the end; empty: no shares
  std::vector<TileItem> tiles;
  std::vector<MergeRow> merge;
  int n_parts = 0, chunk = 0, longest = 0;
};

// Partials that tile items may leave in all, beyond one per token: two rounds of tile items on every SM.
inline long long tile_slots(const SegmentGeometry& g, int sms) {
  return static_cast<long long>((2 * sms + g.kv_heads - 1) / g.kv_heads) * (g.group() <= kTileRows ? g.tile_tokens() + 2 : 0);
}
inline int own_extra(const SegmentGeometry& g) { return decode_max_extra(g.kv_heads); }
// Most partials of a step: prefix steps leave one of each kind per token even when nothing is cut.
inline long long most_parts(const SegmentGeometry& g, int sms, bool prefix) {
  return (prefix ? 2ll * g.n_tokens : 0ll) + tile_slots(g, sms) + 2ll * own_extra(g);
}

// In how many ranges each segment's keys are cut.  One SM works an item off in about one unit per key tile and row
// group (less than two for both groups) and kItemCost for its start and end; a range more costs its partials.  The
// cut that ends first by that account, over all item lengths.
inline void cut_segments(std::vector<Segment>& segs, const SegmentGeometry& g, int sms, long long slots, bool prefix) {
  constexpr double kItemCost = 2.0, kTwoGroups = 1.5, kMerge = 3.0;
  int longest = 0;
  for (const Segment& s : segs) longest = std::max(longest, (s.kv_len + kTileKeys - 1) / kTileKeys);
  double best = -1;
  int best_len = longest;
  for (int n = 1; n <= 64 && n <= longest; ++n) {
    const int len = (longest + n - 1) / n;
    double total = 0, most = 0;
    long long used = 0;
    for (const Segment& s : segs) {
      const int kt = (s.kv_len + kTileKeys - 1) / kTileKeys, c = (kt + len - 1) / len, per = (kt + c - 1) / c;
      const long long full = s.n_tok / g.tile_tokens(), rest = (s.n_tok - full * g.tile_tokens()) * static_cast<long long>(g.group());
      const long long rows = static_cast<long long>(s.n_tok) * g.group();
      const bool halves = rest > 0 && rest <= kTileRows / 2 && (prefix || c > 1) && per > 1;
      if (prefix || c > 1) used += s.n_tok * static_cast<long long>(c * (rows <= kTileRows / 2 && per > 1 ? 2 : 1));
      const double two = kItemCost + kTwoGroups * per, one = kItemCost + (halves ? 0.55 : 1.0) * per;
      total += g.kv_heads * c * (full * two + (rest > kTileRows / 2 ? two : rest > 0 ? one : 0.0));
      most = std::max(most, full > 0 || rest > kTileRows / 2 ? two : one);
    }
    if (used > slots) continue;
    // longest items first, dealt in turn: at worst an even share and most of the last item
    const double even = total / sms, time = std::max(most, even > most ? even + 0.5 * most : even) + (n > 1 && !prefix ? kMerge : 0.0) +
                                            4.0 * static_cast<double>(used) * g.q_heads * g.head_dim / 1e6;
    if (best < 0 || time < best) { best = time; best_len = len; }
  }
  for (Segment& s : segs) {
    const int kt = (s.kv_len + kTileKeys - 1) / kTileKeys;
    s.chunks = best < 0 ? 1 : (kt + best_len - 1) / best_len;
    s.slots = 0;
  }
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

// Puts everything together.  out.rows holds the segments' tokens already; `empty`: tokens without keys.
inline void list_segments(std::vector<Segment>& segs, const std::vector<OwnRange>& own, const std::vector<int>& empty, const SegmentGeometry& g,
                          int sms, bool prefix, SegmentLists& out) {
  cut_segments(segs, g, sms, tile_slots(g, sms) + (prefix ? g.n_tokens : 0), prefix);
  std::vector<int> pieces;
  cut_own(own, g, own_extra(g), out, pieces);
  // the tiles, with the partials of each of their tokens numbered from 0
  const int group = g.group();
  for (Segment& s : segs) {
    const int kt = (s.kv_len + kTileKeys - 1) / kTileKeys, per = (kt + s.chunks - 1) / s.chunks;
    s.chunks = (kt + per - 1) / per;
    const long long rows = static_cast<long long>(s.n_tok) * group;
    const bool partial = prefix || s.chunks > 1;
    // all of a segment's rows leave the same number of partials: only one that fits a single group is halved
    const bool halves = partial && rows <= kTileRows / 2 && per > 1;
    s.slots = partial ? s.chunks * (halves ? 2 : 1) : 0;
    for (int c = 0; c < s.chunks; ++c) {
      const int begin = c * per * kTileKeys, len = std::min(per * kTileKeys, s.kv_len - begin);
      const bool two = halves && len > kTileKeys;
      for (int t = 0; t < s.n_tok; t += g.tile_tokens()) {
        const int n = std::min(g.tile_tokens(), s.n_tok - t), tok0 = s.tok0 + t;
        const bool row = out.rows[tok0 + n - 1].token - out.rows[tok0].token == n - 1;      // (they ascend)
        out.tiles.push_back(TileItem{tok0, n, begin, len, partial ? c * (halves ? 2 : 1) : -1,
                                     (row ? kConsecutive : 0) | (halves && !two ? kEmptySecond : 0), two ? 1 : 0, 0});
      }
    }
  }
  auto cost = [group](const TileItem& t) {
    const int kt = (t.kv_len + kTileKeys - 1) / kTileKeys;
    return t.halves ? (kt + 1) / 2 * 2 : kt * (t.n_tok * group > kTileRows / 2 ? 3 : 2);
  };
  std::stable_sort(out.tiles.begin(), out.tiles.end(), [&](const TileItem& x, const TileItem& y) { return cost(x) > cost(y); });
  // partial slots: a token's tiles' first, then its own pieces'
  std::vector<int> own_of(g.n_tokens, -1), base(own.size(), -1);
  for (size_t i = 0; i < own.size(); ++i) own_of[own[i].token] = static_cast<int>(i);
  for (const Segment& s : segs)
    for (int t = 0; t < s.n_tok; ++t) {
      RowToken& r = out.rows[s.tok0 + t];
      const int o = own_of[r.token], n = s.slots + (o >= 0 ? pieces[o] : 0);
      r.part_base = out.n_parts;
      if (s.slots == 0 && o < 0) continue;
      if (o >= 0) base[o] = out.n_parts + s.slots;
      out.merge.push_back(MergeRow{r.token, out.n_parts, n, 0});
      out.n_parts += n;
    }
  for (size_t i = 0; i < own.size(); ++i)
    if (base[i] < 0 && pieces[i] > 1) {
      base[i] = out.n_parts;
      out.merge.push_back(MergeRow{own[i].token, out.n_parts, pieces[i], 0});
      out.n_parts += pieces[i];
    }
  for (WorkItem& w : out.items) {
    const int i = w.token;
    w.token = own[i].token;
    w.part = base[i] < 0 ? -1 : base[i] + w.part;
  }
  for (int t : empty) out.merge.push_back(MergeRow{t, 0, 0, 0});
}

}  // namespace pkv
