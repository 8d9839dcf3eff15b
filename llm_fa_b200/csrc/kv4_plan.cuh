// How the attention over the 4-bit cache is spread over a persistent grid.
//
// A unit is one (sequence, key/value head, tile of query rows); its work is a
// list of 32-token tiles. Lengths are known on the device only, so every CTA
// derives its share from them: units are laid side by side on one axis, a unit
// taking kKv4UnitCost + tiles of it (the fixed part stands for what a unit
// costs besides its tiles), and CTA c of `parts` takes the c-th equal range.
// A unit cut by range ends has one piece a CTA; the combine kernel joins them.
// Host code runs the same functions in its tests.
#pragma once
#include "kv4_layout.cuh"

namespace llmfa {

constexpr int kKv4TileTokens = 32;
constexpr int kKv4UnitCost = 4;
// Least cost of a CTA's share: 8 warps, a tile each, and the unit's own.
constexpr int kKv4MinShare = 12;

struct Kv4Split {
  const uint32_t* prefix;  // [batch + 1]: cost of one (head, row tile) of the sequences before b
  int batch;
  int hr;          // heads * row tiles
  long long cost;  // of everything
  int parts;       // CTAs that get a share

  __host__ __device__ int tiles(int b) const {
    return static_cast<int>(prefix[b + 1] - prefix[b]) - kKv4UnitCost;
  }
  __host__ __device__ long long bound(int c) const { return cost * c / parts; }
  // CTA whose range holds point x of the axis.
  __host__ __device__ int owner(long long x) const {
    return static_cast<int>(((x + 1) * parts - 1) / cost);
  }
  // Start of unit (b, hr) on the axis.
  __host__ __device__ long long start(int b, int i) const {
    return static_cast<long long>(prefix[b]) * hr + static_cast<long long>(i) * (prefix[b + 1] - prefix[b]);
  }
};

// Tiles of a sequence of n slots; at least one, so that every unit has an owner.
__host__ __device__ inline int kv4_tiles(int n) {
  const int t = static_cast<int>((static_cast<long long>(n) + kKv4TileTokens - 1) / kKv4TileTokens);
  return t > 0 ? t : 1;
}

__host__ __device__ inline Kv4Split kv4_split(const uint32_t* prefix, int batch, int hr, int ctas) {
  Kv4Split s{prefix, batch, hr, static_cast<long long>(prefix[batch]) * hr, 1};
  const long long most = s.cost / kKv4MinShare;
  s.parts = static_cast<int>(most < 1 ? 1 : most < ctas ? most : ctas);
  return s;
}

// The segments of one CTA, in order: unit (b, i), its tiles [lo, hi).
struct Kv4Segment {
  int b, i, lo, hi, tiles;
  long long at, end;  // start of the unit, end of the CTA's range

  // Moves to the next unit that has tiles in the range; false at its end.
  __host__ __device__ bool settle(const Kv4Split& s, long long from) {
    while (at < end) {
      tiles = s.tiles(b);
      const long long l = from - at - kKv4UnitCost, h = end - at - kKv4UnitCost;
      lo = static_cast<int>(l < 0 ? 0 : l);
      hi = static_cast<int>(h < tiles ? h : tiles);
      if (lo < hi) return true;
      step(s);
    }
    return false;
  }
  __host__ __device__ void step(const Kv4Split& s) {
    at += tiles + kKv4UnitCost;
    if (++i == s.hr) {
      i = 0;
      ++b;
    }
  }
  __host__ __device__ bool first(const Kv4Split& s, int c) {
    const long long from = s.bound(c);
    end = s.bound(c + 1);
    int l = 0, h = s.batch - 1;  // the last sequence that starts at or before `from`
    while (l < h) {
      const int m = (l + h + 1) >> 1;
      if (static_cast<long long>(s.prefix[m]) * s.hr <= from) l = m; else h = m - 1;
    }
    b = l;
    const long long rest = from - static_cast<long long>(s.prefix[b]) * s.hr;
    i = static_cast<int>(rest / (s.prefix[b + 1] - s.prefix[b]));
    at = s.start(b, i);
    return settle(s, from);
  }
  __host__ __device__ bool next(const Kv4Split& s) {
    step(s);
    return settle(s, at);
  }
};

// CTAs that hold a unit: the first, and how many.
struct Kv4Pieces {
  int first, count;
};
__host__ __device__ inline Kv4Pieces kv4_pieces(const Kv4Split& s, long long at, int tiles) {
  const int a = s.owner(at + kKv4UnitCost), z = s.owner(at + kKv4UnitCost + tiles - 1);
  return {a, z - a + 1};
}
// Partial-result slot of piece k of a unit: a CTA's last segment goes on in the
// next CTA, its first may have begun in the one before.
__host__ __device__ inline int kv4_slot(int first, int k) { return 2 * (first + k) + (k == 0 ? 1 : 0); }

}  // namespace llmfa
