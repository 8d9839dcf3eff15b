// Host run of the overlap test of strided views (kv4_views.h) against marks in an array.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../llm_fa_b200/csrc/kv4_views.h"

using namespace llmfa;

static bool marked(const Kv4View& a, const Kv4View* b) {
  std::vector<char> mem(1 << 20, 0);
  for (int pass = 0; pass < (b == nullptr ? 1 : 2); ++pass) {
    const Kv4View& v = pass == 0 ? a : *b;
    for (int64_t i = 0; i < v.size[0]; ++i)
      for (int64_t j = 0; j < v.size[1]; ++j)
        for (int64_t k = 0; k < v.size[2]; ++k)
          for (int c = 0; c < 128; ++c) {
            char& m = mem[v.at / 2 + i * v.stride[0] + j * v.stride[1] + k * v.stride[2] + c];
            if (b == nullptr ? m != 0 : pass == 1 && m != 0) return true;
            if (pass == 0) m = 1;
          }
  }
  return false;
}

static int failed(const char* what) {
  std::printf("failed: %s\n", what);
  return 1;
}

int main() {
  unsigned seed = 1;
  auto rnd = [&](int n) { return static_cast<int>((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  int yes = 0, no = 0, self = 0;
  for (int it = 0; it < 6000; ++it) {
    Kv4View v[2];
    for (auto& x : v) {
      x.at = 16 * rnd(it % 2 ? 64 : 4096);
      const int wide = rnd(2) ? 128 : 8 * (1 + rnd(48));
      int64_t s[3];
      int64_t inner = wide;
      for (int d = 0; d < 3; ++d) {
        x.size[d] = 1 + rnd(5);
        s[d] = rnd(4) == 0 ? 8 * (1 + rnd(200)) : inner;  // nested, or anything
        inner = s[d] * (x.size[d] + rnd(2));
      }
      const int turn = rnd(3);
      for (int d = 0; d < 3; ++d) x.stride[d] = s[(d + turn) % 3];
      int64_t size[3] = {x.size[0], x.size[1], x.size[2]};
      for (int d = 0; d < 3; ++d) x.size[d] = size[(d + turn) % 3];
    }
    const bool want = marked(v[0], &v[1]);
    if (Kv4Meeting(v[0], &v[1]).found() != want || Kv4Meeting(v[1], &v[0]).found() != want)
      return failed("two views");
    const bool twice = marked(v[0], nullptr);
    if (Kv4Meeting(v[0], nullptr).found() != twice) return failed("one view");
    (want ? yes : no)++;
    self += twice;
  }
  if (yes < 500 || no < 500 || self < 200) return failed("too few of a kind");
  // large ones: slices of a fused tensor, of any layout, are told apart in few steps
  const int64_t B = 4096, T = 1 << 20, H = 96;
  const Kv4View q{1 << 20, {T * 3 * H * 128, 3 * H * 128, 128}, {B, T, H}};
  Kv4View k = q;
  k.at += 2 * H * 128;
  if (Kv4Meeting(q, &k).found() || Kv4Meeting(q, nullptr).found()) return failed("fused");
  k.at -= 16;
  if (!Kv4Meeting(q, &k).found()) return failed("fused, 8 elements early");
  const Kv4View even{1 << 20, {T * H * 256, H * 256, 256}, {B, T, H}};
  Kv4View odd{(1 << 20) + 256, {256, H * 256, T * H * 256}, {H, T, B}};
  if (Kv4Meeting(even, &odd).found()) return failed("interleaved");
  std::printf("ok\n");
  return 0;
}
