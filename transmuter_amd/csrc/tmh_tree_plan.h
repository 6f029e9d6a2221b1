// What the rows of a drafted step see of a paged cache, and how attention over it is shared out: whole numbers only, the
// same on the host (whose tests go over them) and on the device.
#pragma once

#include "tmh_paged_plan.h"

namespace tmh {

// One sequence of a drafted step: rows [row, row + nodes) of the step are the last `nodes` of its tokens, node i the token
// prefix + i (with fewer tokens in the cache than nodes the first nodes have none, and prefix is negative). Its columns, each
// query head of one kv head for each node, go to tiles of `columns`. Units (`unit_tokens` tokens each, counted from token 0)
// hold what any of its rows may see; a window leaves the units before it out.
struct Draft {
  int row, nodes, prefix, end, unit, units, tiles;
};
TMH_HD Draft draft_of(int32_t start, int32_t stop, int64_t rows, int32_t length, int64_t most, int window, int unit_tokens, int group,
                      int columns) {
  Draft d;
  const int64_t n = length < 0 ? 0 : length < most ? length : most;
  const int64_t from = start < 0 ? 0 : start < rows ? start : rows, to = stop < from ? from : stop < rows ? stop : rows;
  d.row = static_cast<int>(from);
  d.nodes = static_cast<int>(to - from);
  d.end = static_cast<int>(n);
  d.prefix = d.end - d.nodes;
  const int begin = window > 0 && d.prefix > window ? d.prefix - window : 0;
  d.unit = begin / unit_tokens;
  d.units = d.nodes > 0 && n > 0 ? static_cast<int>((n + unit_tokens - 1) / unit_tokens) - d.unit : 0;
  d.tiles = static_cast<int>((static_cast<int64_t>(d.nodes) * group + columns - 1) / columns);
  return d;
}

// Which of the 32 tokens from node `first` on (negative: tokens ahead of the nodes, all of which count) a row's tree has:
// bit j % 64 of word j / 64 is node j.
TMH_HD uint32_t tree_bits(const uint64_t* words, int count, int first) {
  if (first <= -32) return ~0u;
  if (first < 0) return static_cast<uint32_t>((count > 0 ? words[0] : 0) << -first) | ((1u << -first) - 1);
  const int at = first >> 6, shift = first & 63;
  const uint64_t low = at < count ? words[at] >> shift : 0;
  const uint64_t high = shift > 32 && at + 1 < count ? words[at + 1] << (64 - shift) : 0;
  return static_cast<uint32_t>(low | high);
}
// The same in a chain: node `node` has those up to itself.
TMH_HD uint32_t chain_bits(int node, int first) {
  const int n = node - first + 1;
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
}
// The 32 tokens from `first` on that are not before `begin`.
TMH_HD uint32_t from_bits(int begin, int first) {
  const int n = begin - first;
  return n <= 0 ? ~0u : n >= 32 ? 0u : ~0u << n;
}

// The first token that a row sees with a window of at least 1: the last `window` of its tokens, those of its tree being the
// last, count.
TMH_HD int tree_begin(const uint64_t* words, int count, int prefix, int nodes, int window) {
  const int none = prefix < 0 ? -prefix : 0;  // nodes that have no token
  int left = window;
  for (int w = (nodes + 63) / 64 - 1; w >= 0; --w) {
    if (w >= count) continue;
    uint64_t bits = words[w];
    if (nodes - 64 * w < 64) bits &= (uint64_t{1} << (nodes - 64 * w)) - 1;
    if (none > 64 * w) bits = none - 64 * w < 64 ? bits & ~uint64_t{0} << (none - 64 * w) : 0;
    int n = __builtin_popcountll(bits);
    if (n >= left) {
      for (; n > left; --n) bits &= bits - 1;
      return prefix + 64 * w + __builtin_ctzll(bits);
    }
    left -= n;
  }
  return prefix > left ? prefix - left : 0;
}
TMH_HD int chain_begin(int node, int prefix, int window) {
  const int end = prefix + node + 1;
  return end > window ? end - window : 0;
}

// How the work is shared out. An item, one kv head's tile of columns over all units of its sequence, counts as kItem units more
// than it has, ahead of them: the way in (its queries, masks and first rows, one after another from memory) and out. All items lie
// in order and are cut into equal runs, one a worker, which so may begin or end within what only counts. What a worker has of an
// item that it does not have whole is a part, of which it keeps two at most: in place 2 w one that does not begin the item, in
// 2 w + 1 one that does. (With kItem 0, 4 and 8, in us: 16 x 16 nodes over 4000 bf16 58, 51, 52; 8 x 32 54, 42, 43; 4 x 8 over 2000 f32
// 54, 41, 41; one of 64 over 131072, where items are long, 278, 297, 298.)
constexpr uint32_t kItem = 4;
TMH_HD uint32_t work_of(const Draft& d) {  // of one kv head
  return d.units ? (static_cast<uint32_t>(d.units) + kItem) * static_cast<uint32_t>(d.tiles) : 0;
}
// The units [from, to) of an item whose work begins at `first` that lie in [at, stop) (none: from >= to).
struct Share {
  uint32_t from, to;
};
TMH_HD Share share_of(uint32_t first, uint32_t units, uint32_t at, uint32_t stop) {
  const uint32_t begin = first + kItem, end = begin + units;
  const uint32_t from = at > begin ? at : begin, to = stop < end ? stop : end;
  return {from - begin, to > begin ? to - begin : 0};
}
TMH_HD uint32_t place_of_part(uint32_t worker, bool begins) { return 2 * worker + (begins ? 1 : 0); }
// The parts of an item: those of the workers `from` .. `from + count - 1` (count 1: the worker has it whole).
struct TreeParts {
  uint32_t from, count;
};
TMH_HD TreeParts tree_parts(uint32_t first, uint32_t units, uint32_t per) {
  const uint32_t from = (first + kItem) / per;
  return {from, (first + kItem + units - 1) / per - from + 1};
}

}  // namespace tmh
