// How the attention over the 4-bit cache is spread over the GPU.
//
// A unit is one (sequence, key/value head, tile of query rows); its work is a
// list of 32-token tiles. The workers are the warps of a persistent grid: a
// warp needs no other to go through its tokens, so nothing waits where a unit
// begins or ends. Lengths are known on the device only, so every worker derives
// its share from them: units are laid side by side on one axis, a unit taking
// kKv4UnitCost + tiles of it (the fixed part stands for what a unit costs
// besides its tiles), and worker w takes the w-th range of `share`. A unit cut
// by range ends has one piece a worker; the combine kernel joins them. Host
// code runs the same functions in its tests.
#pragma once
#include "kv4_layout.cuh"

namespace llmfa {

constexpr int kKv4TileTokens = 32;
constexpr int kKv4UnitCost = 1;
// Least share: one tile. A tile takes a lone warp 1.2 us, more than joining its piece (1 x 1000
// tokens, 8 heads: 12.4 us, with two tiles a worker 14.4, with three 16.4).
constexpr int kKv4MinShare = kKv4UnitCost + 1;

struct Kv4Split {
  const uint32_t* prefix;  // [batch + 1]: cost of one (head, row tile) of the sequences before b
  int batch;
  int hr;           // heads * row tiles
  long long cost;   // of everything
  long long share;  // of a worker
  double inverse;   // 1 / share

  __host__ __device__ int tiles(int b) const {
    return static_cast<int>(prefix[b + 1] - prefix[b]) - kKv4UnitCost;
  }
  // Worker whose range holds point x of the axis. The product is off by less than one, and the
  // comparisons put it right: a 64-bit division costs a hundred instructions.
  __host__ __device__ int owner(long long x) const {
    long long w = static_cast<long long>(static_cast<double>(x) * inverse);
    if (w * share > x) --w;
    if ((w + 1) * share <= x) ++w;
    return static_cast<int>(w);
  }
  // Start of unit (b, i) on the axis.
  __host__ __device__ long long start(int b, int i) const {
    return static_cast<long long>(prefix[b]) * hr + static_cast<long long>(i) * (prefix[b + 1] - prefix[b]);
  }
};

// Tiles of a sequence of n slots; at least one, so that every unit has an owner.
__host__ __device__ inline int kv4_tiles(int n) {
  const int t = static_cast<int>((static_cast<long long>(n) + kKv4TileTokens - 1) / kKv4TileTokens);
  return t > 0 ? t : 1;
}

__host__ __device__ inline Kv4Split kv4_split(const uint32_t* prefix, int batch, int hr, int workers) {
  const long long cost = static_cast<long long>(prefix[batch]) * hr;
  const long long even = (cost + workers - 1) / workers;
  const long long share = even < kKv4MinShare ? kKv4MinShare : even;
  return Kv4Split{prefix, batch, hr, cost, share, 1.0 / static_cast<double>(share)};
}

// The segments of one worker, in order: unit (b, i), its tiles [lo, hi).
struct Kv4Segment {
  int b, i, lo, hi, tiles;
  long long at, end;  // start of the unit, end of the worker's range

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
  __host__ __device__ bool first(const Kv4Split& s, int worker) {
    const long long from = worker * s.share;
    end = from + s.share < s.cost ? from + s.share : s.cost;
    if (from >= end) return false;
    int l = 0, h = s.batch - 1;  // the last sequence that starts at or before `from`
    while (l < h) {
      const int m = (l + h + 1) >> 1;
      if (static_cast<long long>(s.prefix[m]) * s.hr <= from) l = m; else h = m - 1;
    }
    b = l;
    const uint32_t unit = s.prefix[b + 1] - s.prefix[b];
    const long long rest = from - static_cast<long long>(s.prefix[b]) * s.hr;
    i = rest >> 32 == 0 ? static_cast<int>(static_cast<uint32_t>(rest) / unit)
                        : static_cast<int>(rest / unit);
    at = s.start(b, i);
    return settle(s, from);
  }
  __host__ __device__ bool next(const Kv4Split& s) {
    step(s);
    return settle(s, at);
  }
  __host__ __device__ bool whole() const { return lo == 0 && hi == tiles; }
};

// Workers that hold a unit: the first, and how many.
struct Kv4Pieces {
  int first, count;
};
__host__ __device__ inline Kv4Pieces kv4_pieces(const Kv4Split& s, long long at, int tiles) {
  const int a = s.owner(at + kKv4UnitCost), z = s.owner(at + kKv4UnitCost + tiles - 1);
  return {a, z - a + 1};
}
// Partial-result slot of piece k of a unit: a worker's last segment goes on in the next worker,
// its first may have begun in the one before.
__host__ __device__ inline int kv4_slot(int first, int k) { return 2 * (first + k) + (k == 0 ? 1 : 0); }

}  // namespace llmfa
