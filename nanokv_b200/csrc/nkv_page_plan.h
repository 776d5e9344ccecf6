// What the paged 16-bit cache takes from memory that the host does not see, and how its attention is dealt out to thread
// blocks.  Plain C++, so that it can be checked without a GPU.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define NKV_PAGE_INLINE __host__ __device__ __forceinline__
#else
#define NKV_PAGE_INLINE inline
#endif

namespace nkv {
namespace page {

NKV_PAGE_INLINE int least(int a, int b) { return a < b ? a : b; }
NKV_PAGE_INLINE int most(int a, int b) { return a > b ? a : b; }

// Settled tokens of a sequence, pending ones that the call names, and those of them that the table has room for.
struct Extent { int length, count, there; };
NKV_PAGE_INLINE Extent extent_in(int length, int count, int tokens, int room, bool& bad) {
  Extent e;
  e.length = least(most(length, 0), room);
  e.count = least(most(count, 0), tokens);
  e.there = least(e.count, room - e.length);
  bad = e.length != length || e.count != count || e.there != e.count;
  return e;
}

NKV_PAGE_INLINE uint32_t first_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

enum Sight { SEES_ALL, SEES_CAUSAL, SEES_TREE };

// Which of tokens first .. first + 31 query t sees, as bits: all settled ones and, of the pending ones, those of its mask.
// `word(w)`: word w of the query's mask, 0 outside it.
template <class Word>
NKV_PAGE_INLINE uint32_t sight_bits(int sight, const Extent& e, int t, int first, Word word) {
  const int j = first - e.length;
  if (j <= -32) return 0xFFFFFFFFu;
  uint32_t bits;
  if (sight == SEES_ALL) {
    bits = first_bits(e.there - j);
  } else if (sight == SEES_CAUSAL) {
    bits = first_bits(least(t + 1, e.there) - j);
  } else {
    const int w = j >= 0 ? j / 32 : -1, shift = j - 32 * w;
    const uint32_t lo = word(w), hi = word(w + 1);
    bits = (shift ? lo >> shift | hi << (32 - shift) : lo) & first_bits(e.there - j);
  }
  return j < 0 ? bits | first_bits(-j) : bits;
}

// tokens from the first on that query t sees all of
NKV_PAGE_INLINE int sees_all_before(int sight, const Extent& e, int t) {
  if (t >= e.count) return 0;
  return e.length + (sight == SEES_TREE ? 0 : sight == SEES_CAUSAL ? least(t + 1, e.there) : e.there);
}

// ---- attention: units of query rows of a kv head, tiles of tokens -------------------------------------------------
constexpr int TOK = 128;             // tokens of a tile
constexpr int MOST_SEQUENCES = 96;   // of one launch; longer batches are cut

struct Shape { int sight, group, rows, unit, units, kv_heads; };   // rows of a kv head, rows of a unit, units

// tiles that rows [r0, r0 + n) need
NKV_PAGE_INLINE int tiles_seen(const Shape& s, const Extent& e, int r0, int n) {
  const int r1 = least(s.rows, r0 + n) - 1;
  if (r1 < r0 || r0 / s.group >= e.count) return 0;
  const int seen = sees_all_before(s.sight == SEES_TREE ? SEES_ALL : s.sight, e, least(r1 / s.group, e.count - 1));
  return (seen + TOK - 1) / TOK;
}

// A unit costs a run as much as PIECE_TILES tiles on top of its own: its queries' way in and its rows' way out (costs of 2 / 3 / 5 / 7 / 9,
// over four states in turn, us: 2 x 4,095 causal queries x 32 heads fp16 375 / 371 / 352 / 357 / 361, bf16 372 / 368 / 348 / 354 / 358; one token each of
// 31 sequences of up to 2,138 x 320 heads 197 / 189 / 180 / 174 / 177, of 32 of up to 4,096 x 32 heads over 8 77 / 73 / 70 / 69 / 71; 32 trees of 16 nodes
// 240 / 236 / 235 / 238 / 238, 8 of 63 nodes over 64-wide heads 56 / 55 / 54 / 54 / 56; 99,840 tokens x 40 heads 336 to 339 with each).
constexpr uint32_t PIECE_TILES = 5;
NKV_PAGE_INLINE uint32_t cost_of(int tiles) { return tiles > 0 ? tiles + PIECE_TILES : 0; }

// The list of tiles: sequence by sequence, kv head by kv head, unit by unit, with PIECE_TILES places ahead of a unit's.  It is cut into
// equal runs, of which thread block i takes the i-th, and in further rounds the (blocks + i)-th and so on: blocks that work at the same
// time then work on neighbouring parts of the list, whose keys and values the units of a kv head share in the L2 cache.
struct Plan {
  const uint32_t* start;             // [sequences + 1]
  const Extent* extents;
  int sequences;
  uint32_t run, longer;              // places of a run; the first `longer` have one more
  NKV_PAGE_INLINE void deal(int runs) {
    run = start[sequences] / runs;
    longer = start[sequences] % runs;
  }
  NKV_PAGE_INLINE uint32_t first_of(uint32_t i) const { return i * run + (i < longer ? i : longer); }
  NKV_PAGE_INLINE uint32_t run_of(uint32_t g) const {
    const uint32_t edge = longer * (run + 1);
    return g < edge ? g / (run + 1) : longer + (g - edge) / run;
  }
};

struct Piece {                        // a unit, or a run's part of one
  int b, h, unit, tile0, nt, whole;   // tiles tile0 .. tile0 + nt - 1; whole: all the unit has
};

// Rounds of a call whose units read `bytes` of keys and values: as few as keep what one round reads within FITS, as long as a run
// has `least` places.
constexpr uint64_t FITS = 64ull << 20;
NKV_PAGE_INLINE int rounds_of(uint64_t bytes, uint32_t places, int blocks, int least, int most_rounds) {
  int rounds = 1;
  while (rounds < most_rounds && bytes > FITS * rounds && places / blocks / (rounds + 1) >= static_cast<uint32_t>(least)) ++rounds;
  return rounds;
}
// Of the counts that let a round read between FITS and twice that (L2 holds 126 MB), the one whose runs come closest to a whole number
// of runs a unit: units of a kv head then start and end together and go in step.
NKV_PAGE_INLINE int rounds_for(uint64_t bytes, uint32_t places, uint32_t units, int blocks, int least, int most_rounds) {
  const int most = rounds_of(bytes, places, blocks, least, most_rounds);
  int best = 0;
  uint32_t off = UINT32_MAX;
  for (int rounds = rounds_of(bytes / 2, places, blocks, least, most_rounds); rounds <= most; ++rounds) {
    const uint32_t runs = static_cast<uint32_t>(rounds) * blocks, over = runs % units;
    const uint32_t away = runs < units || units - over < over ? units - over : over;
    if (away < off) {
      off = away;
      best = rounds;
    }
  }
  return best;
}

// The pieces of one run in order.
struct Walk {
  uint32_t g, end;
  int b, h, unit, tiles;              // the unit that g lies in, its tiles
  uint32_t at;                        // places of the unit before g
  NKV_PAGE_INLINE int tiles_of(const Plan& p, const Shape& s) const { return tiles_seen(s, p.extents[b], unit * s.unit, s.unit); }
  NKV_PAGE_INLINE Walk(const Plan& p, const Shape& s, int which) {
    g = p.first_of(which);
    end = p.first_of(which + 1);
    b = h = unit = tiles = 0;
    at = 0;
    if (g >= end) return;
    int lo = 0, hi = p.sequences - 1;   // the last sequence that starts at or before g, and has places
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.start[mid] <= g) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const uint32_t per_head = (p.start[b + 1] - p.start[b]) / s.kv_heads;
    at = g - p.start[b];
    h = static_cast<int>(at / per_head);
    at -= h * per_head;
    while (at >= cost_of(tiles = tiles_of(p, s))) {
      at -= cost_of(tiles);
      ++unit;
    }
  }
  NKV_PAGE_INLINE bool next(const Plan& p, const Shape& s, Piece& out) {
    uint32_t from, to;
    do {
      if (g >= end) return false;
      while (at >= cost_of(tiles)) {   // on to the next unit that has tiles
        at = 0;
        if (++unit == s.units) {
          unit = 0;
          if (++h == s.kv_heads) {
            h = 0;
            do ++b; while (p.start[b + 1] == p.start[b]);
          }
        }
        tiles = tiles_of(p, s);
      }
      from = at;
      to = cost_of(tiles) < at + (end - g) ? cost_of(tiles) : at + (end - g);
      g += to - from;
      at = to;
    } while (to <= PIECE_TILES);       // (the run's end, ahead of the unit's tiles)
    out.b = b;
    out.h = h;
    out.unit = unit;
    out.tile0 = static_cast<int>((from > PIECE_TILES ? from : PIECE_TILES) - PIECE_TILES);
    out.nt = static_cast<int>(to - PIECE_TILES) - out.tile0;
    out.whole = out.nt == tiles;
    return true;
  }
};

// The pieces of a thread block, run by run; every role of it makes the same tour.
struct Tour {
  int run, step, runs;                // the run at hand, from one of the block's to the next, all of them
  Walk walk;
  NKV_PAGE_INLINE Tour(const Plan& p, const Shape& s, int block, int blocks, int rounds)
      : run(block), step(blocks), runs(blocks * rounds), walk(p, s, block) {}
  NKV_PAGE_INLINE bool next(const Plan& p, const Shape& s, Piece& out) {
    while (!walk.next(p, s, out)) {
      if (run + step >= runs) return false;
      run += step;
      walk = Walk(p, s, run);
    }
    return true;
  }
  // the run that has the last tile of the unit at hand
  NKV_PAGE_INLINE int last_run(const Plan& p) const { return static_cast<int>(p.run_of(walk.g + cost_of(walk.tiles) - walk.at - 1)); }
};

}  // namespace page
}  // namespace nkv
