// Host run of the 4-bit attention's work split (kv4_plan.cuh): every tile of every unit is in
// exactly one worker's segments, pieces are found again with distinct slots, shares are even.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>

#include "../../llm_fa_b200/csrc/kv4_plan.cuh"

using namespace llmfa;

#define CHECK(c) \
  do { \
    if (!(c)) { \
      std::printf("failed: %s (line %d)\n", #c, __LINE__); \
      std::exit(1); \
    } \
  } while (0)

static void run(const std::vector<int>& lens, int hr, int ctas) {
  const int B = static_cast<int>(lens.size());
  std::vector<uint32_t> prefix(B + 1, 0);
  for (int b = 0; b < B; ++b) prefix[b + 1] = prefix[b] + kv4_tiles(lens[b]) + kKv4UnitCost;
  const Kv4Split s = kv4_split(prefix.data(), B, hr, ctas);
  CHECK(s.share >= kKv4MinShare && s.share * ctas >= s.cost);
  CHECK(s.share == kKv4MinShare || (s.share - 1) * ctas < s.cost);
  std::map<std::pair<int, int>, std::vector<std::pair<int, Kv4Segment>>> pieces;
  for (int c = 0; c < ctas; ++c) {
    Kv4Segment g{};
    for (bool ok = g.first(s, c); ok; ok = g.next(s)) {
      CHECK(g.b >= 0 && g.b < B && g.i >= 0 && g.i < hr && g.tiles == kv4_tiles(lens[g.b]));
      CHECK(0 <= g.lo && g.lo < g.hi && g.hi <= g.tiles && g.at == s.start(g.b, g.i));
      pieces[{g.b, g.i}].push_back({c, g});
    }
  }
  CHECK(static_cast<int>(pieces.size()) == B * hr);
  std::set<int> slots;
  for (auto& [unit, list] : pieces) {
    int at = 0;
    const Kv4Segment& g = list[0].second;
    const Kv4Pieces p = kv4_pieces(s, g.at, g.tiles);
    CHECK(p.count == static_cast<int>(list.size()) && p.first == list[0].first);
    for (int k = 0; k < p.count; ++k) {
      CHECK(list[k].first == p.first + k && list[k].second.lo == at);
      at = list[k].second.hi;
      if (p.count > 1) {
        const int slot = kv4_slot(p.first, k);
        CHECK(slot >= 0 && slot < 2 * ctas && slots.insert(slot).second);
        CHECK(!list[k].second.whole());
        // the slot that the worker itself derives from its segment
        CHECK(slot == 2 * list[k].first + (list[k].second.lo == 0 ? 1 : 0));
      }
    }
    CHECK(at == g.tiles);
  }
}

int main() {
  unsigned seed = 1;
  auto rnd = [&](int n) { return static_cast<int>((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  for (int ctas : {1, 2, 7, 148, 2368}) {
    run({0}, 1, ctas);
    run({1}, 1, ctas);
    run({131071}, 8, ctas);
    run({1000}, 8, ctas);
    run({31, 32, 33, 0, 0, 64}, 5, ctas);
    for (int k = 0; k < 60; ++k) {
      std::vector<int> lens(1 + rnd(k % 10 == 0 ? 600 : 20));
      const int top = 1 << rnd(15);
      for (int& n : lens) n = rnd(4) == 0 ? 0 : rnd(top + 1);
      run(lens, 1 + rnd(40), ctas);
    }
  }
  // costs past 32 bits
  std::vector<int> lens(300, (1 << 28));
  const int B = 300;
  std::vector<uint32_t> prefix(B + 1, 0);
  for (int b = 0; b < B; ++b) prefix[b + 1] = prefix[b] + 6000000u + kKv4UnitCost;
  const Kv4Split s = kv4_split(prefix.data(), B, 1024, 296);
  CHECK(s.cost > (1ll << 40));
  for (long long x : {0ll, 1ll, s.share - 1, s.share, s.share + 1, 17 * s.share - 1, 17 * s.share, s.cost - 1})
    CHECK(s.owner(x) == x / s.share);
  long long sum = 0;
  for (int c = 0; c < 296; ++c) {
    Kv4Segment g{};
    long long n = 0;
    for (bool ok = g.first(s, c); ok && n < 10; ok = g.next(s), ++n) sum += g.hi - g.lo > 0;
    CHECK(n == 10);
  }
  std::printf("ok\n");
  return 0;
}
