// The equal shares of packed attention's dK / dV pass (packed_attn.hip), apart from it because the host's tests compile them too: which steps of which
// key tiles a block walks, and where a tile that lies in several shares leaves its sums.
//
// One axis: each key head has `total` units, key tile t's of a head lie at units[t] .. units[t + 1] - 1 of them - OPERANDS for its operands and results,
// then one for each of its steps - and block b takes the `share` units from b * share on.  A tile that is not whole in one share leaves a partial sum:
// slot 2 b + 1 of the block in which it begins, slot 2 b of the others (a block goes on with at most one tile and begins at most one that it does not end).
// `units` is the caller's device memory.  A block's share, and so its slots, come from the numbers that the host sized grid and workspace with, never from
// the table: whatever that holds, no slot lies outside the 2 * blocks of the workspace, a segment's steps are steps of its tile, and every walk ends.
#pragma once

#ifdef __HIP__
#define SHARE_FN __host__ __device__ inline
#else
#define SHARE_FN inline
#endif

namespace {

constexpr int OPERANDS = 2;      // what a dK / dV tile's operands and results count, in steps

SHARE_FN int units_of(const int* units, int t) { return (int)((unsigned)units[t + 1] - (unsigned)units[t]); }      // (wraps where the table is nonsense)
SHARE_FN long at_least(long x, long lo) { return x < lo ? lo : x; }
SHARE_FN long at_most(long x, long hi) { return x > hi ? hi : x; }

struct Place { long pos, end; int kh, ti; };      // the units [pos, end) of a block, the key head and key tile at pos; pos >= end: nothing
SHARE_FN Place place_of(const int* units, int n_tiles, int total, int kv_heads, int share, int block) {
  Place p;
  p.kh = p.ti = 0;
  p.pos = (long)block * share;
  p.end = at_most(p.pos + share, (long)total * kv_heads);      // (at most p.pos behind the last block: the grid is rounded up)
  if (p.pos >= p.end) return p;
  p.kh = (int)(p.pos / total);
  const int u = (int)(p.pos - (long)p.kh * total);
  int lo = 0, hi = n_tiles;      // units[lo] <= u < units[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (units[mid] <= u) lo = mid;
    else hi = mid;
  }
  p.ti = lo;
  return p;
}

struct Segment { int first, last, slot; long next; };      // steps [first, last) of the tile, place of its partial sum (-1: the whole tile), where the walk goes on
// the part of the tile with the units [at, at + mine) and `steps` steps that lies in block `block`'s [pos, end)
SHARE_FN Segment segment_of(long pos, long end, int block, long at, int mine, int steps) {
  Segment s;
  const int u0 = (int)at_most(at_least(pos - at, 0), mine), u1 = (int)at_most(end - at, mine);
  s.slot = u0 > 0 || u1 < mine ? 2 * block + (u0 == 0) : -1;
  s.first = (int)at_most(at_least((long)u0 - OPERANDS, 0), steps);
  s.last = u1 == mine ? steps : (int)at_most(at_least((long)u1 - OPERANDS, s.first), steps);
  s.next = at_least(at + mine, pos + 1);      // (on, whatever the table holds)
  return s;
}

struct Meeting { int first, last; };      // the blocks in which the tile with the units [at, at + mine) has partial sums; first >= last: none
SHARE_FN Meeting meeting_of(long at, int mine, int share, int blocks) {
  Meeting m;
  m.first = (int)at_most(at / share, blocks - 1);
  m.last = (int)at_most((at + mine - 1) / share, blocks - 1);
  if (m.first < 0) m.last = m.first;
  return m;
}

}  // namespace
