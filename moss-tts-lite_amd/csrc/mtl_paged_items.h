// How paged_shared_kernel cuts its work: what items cost, which piece a block falls into, and which
// blocks of an item a piece takes.  Plain C++ without HIP types, so that a host program can walk
// every item of a call.
#pragma once

namespace mtl {

constexpr int kSharedBlock = 128;       // positions of a block
constexpr int kNarrow = 32;             // columns up to which waves take positions, not columns
constexpr int kWide = 64;               // columns of an item, at most

constexpr int blocks_in(int positions) { return (positions + kSharedBlock - 1) / kSharedBlock; }

// What a block of an item costs by its columns, and an item by itself.  An item without blocks is
// not there and has no length in the row of items.
constexpr int block_cost(int columns) { return columns <= 16 ? 3 : columns <= kNarrow ? 4 : 8; }
constexpr int kItemCost = 12;
constexpr int item_cost(int columns, int blocks) {
  return blocks ? kItemCost + blocks * block_cost(columns) : 0;
}

// The cost of `columns` columns over `blocks` blocks, `wide` (a power of two) of them an item.
constexpr int cost_of(int columns, int blocks, int wide) {
  const int rest = columns & (wide - 1);
  return columns / wide * item_cost(wide, blocks) + (rest ? item_cost(rest, blocks) : 0);
}

struct Span {
  int x, y;
};

// The row of all items, cut into pieces that differ by one in length at most.
struct Pieces {
  int each, longer;

  constexpr int start(int piece) const {
    return piece * each + (piece < longer ? piece : longer);
  }
  constexpr int piece_of(int at) const {
    const int head = longer * (each + 1);
    return at < head ? at / (each + 1) : longer + (at - head) / (each > 1 ? each : 1);
  }
  // The first and last piece that an item of `columns` columns and `blocks` blocks from `base` on
  // lies in; (0, -1): it is not there.
  constexpr Span pieces_of(int base, int blocks, int columns) const {
    base += kItemCost;
    return blocks ? Span{piece_of(base), piece_of(base + (blocks - 1) * block_cost(columns))}
                  : Span{0, -1};
  }
};

// The blocks [x, y) of an item that fall into a piece: blocks that begin within [lo, hi).
constexpr Span blocks_within(int base, int blocks, int columns, int lo, int hi) {
  const int each = block_cost(columns);
  base += kItemCost;
  const int x = lo <= base ? 0 : (lo - base + each - 1) / each;
  const int y = hi <= base ? 0 : (hi - base + each - 1) / each;
  return Span{x < blocks ? x : blocks, y < blocks ? y : blocks};
}

// The items of `columns` columns over `blocks` blocks each, from `base` on, which passes over them:
// calls take(first column, columns, blocks [x, y)) for what lies within [lo, hi).
template <int WIDE, class Take>
__attribute__((always_inline)) constexpr void items_within(int& base, int columns, int blocks,
                                                           int lo, int hi, Take&& take) {
  if (blocks == 0) return;
  const int full = item_cost(WIDE, blocks);
  int skip = lo > base ? (lo - base) / full : 0;      // whole items before lo
  if (skip > columns / WIDE) skip = columns / WIDE;
  base += skip * full;
  for (int c = skip * WIDE; c < columns; c += WIDE) {
    const int n = columns - c < WIDE ? columns - c : WIDE;
    const Span b = blocks_within(base, blocks, n, lo, hi);
    if (b.x < b.y) take(c, n, b);
    base += item_cost(n, blocks);
  }
}

}  // namespace mtl
