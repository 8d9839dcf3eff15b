// Whether strided views share memory: a kernel that writes one while it reads or
// writes the other would race. Host code.
#pragma once
#include <algorithm>
#include <cstdint>

namespace llmfa {

// Rows of 128 16-bit values, at multiples of three strides (in elements) from `at`.
struct Kv4View {
  uintptr_t at;  // bytes
  int64_t stride[3], size[3];
};

// Do two rows meet: are there steps t with |distance + sum of t s| < 128? The strides are tried in
// descending order, each t between what the smaller strides can still make up for; the greatest
// common divisor of those decides most layouts at once (slices of one wider tensor). A search that
// would take long says yes.
class Kv4Meeting {
 public:
  // Of a row of `a` with a row of `b`; of two different rows of `a` where b is null.
  Kv4Meeting(const Kv4View& a, const Kv4View* b) {
    for (int j = 0; j < 3; ++j) {
      add(a.stride[j], -(a.size[j] - 1), b == nullptr ? a.size[j] - 1 : 0, b != nullptr);
      if (b != nullptr) add(b->stride[j], 0, b->size[j] - 1, true);
    }
    std::sort(term_, term_ + terms_, [](const Term& x, const Term& y) { return x.s > y.s; });
    bool nested = true;  // every stride passes over all that the smaller ones reach
    for (int j = terms_ - 1; j >= 0; --j) {
      nested &= term_[j].s + low_[j + 1] >= kRow;
      low_[j] = low_[j + 1] + Wide(term_[j].s) * term_[j].lo;
      high_[j] = high_[j + 1] + Wide(term_[j].s) * term_[j].hi;
    }
    // rows start at even addresses, so the distance is whole elements
    const Wide d = b == nullptr ? 0 : (static_cast<Wide>(b->at) - static_cast<Wide>(a.at)) / 2;
    if (b == nullptr ? nested : d + high_[0] <= -kRow || d + low_[0] >= kRow) return;  // most calls
    for (int j = terms_ - 1; j >= 0; --j) gcd_[j] = gcd(term_[j].s, gcd_[j + 1]);
    found_ = search(0, d, b != nullptr);
  }
  bool found() const { return found_; }

 private:
  using Wide = __int128;
  static constexpr int kRow = 128, kMostSteps = 1 << 16;
  struct Term {
    int64_t s, lo, hi;
  };

  static Wide gcd(Wide a, Wide b) {
    while (b != 0) {
      const Wide r = a % b;
      a = b;
      b = r;
    }
    return a;
  }
  static Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0 ? 1 : 0); }  // b > 0

  // Equal strides of two views count as one; of a view's own, steps that make up for one another
  // lead to another row.
  void add(int64_t s, int64_t lo, int64_t hi, bool join) {
    if (lo == hi) return;  // a size of 1: its stride is never used
    for (int j = 0; join && j < terms_; ++j) {
      if (term_[j].s == s) {
        term_[j].lo += lo;
        term_[j].hi += hi;
        return;
      }
    }
    term_[terms_++] = {s, lo, hi};
  }
  bool search(int j, Wide r, bool moved) {
    if (++steps_ > kMostSteps) return true;
    if (r + high_[j] <= -kRow || r + low_[j] >= kRow) return false;
    if (j == terms_) return moved;
    const Wide g = gcd_[j], rest = r - floor_div(r, g) * g;
    if (rest >= kRow && g - rest >= kRow) return false;
    // -kRow < r + s t + [low, high] of the smaller strides < kRow
    const Term& t = term_[j];
    const Wide first = floor_div(-kRow - r - high_[j + 1], t.s) + 1;
    const Wide last = -floor_div(-(kRow - r - low_[j + 1]), t.s) - 1;
    for (Wide i = std::max<Wide>(first, t.lo); i <= std::min<Wide>(last, t.hi); ++i)
      if (search(j + 1, r + i * t.s, moved || i != 0)) return true;
    return false;
  }

  Term term_[6];
  int terms_ = 0, steps_ = 0;
  Wide low_[7] = {}, high_[7] = {}, gcd_[7] = {};
  bool found_ = false;
};

}  // namespace llmfa
