// Host run of the 4-bit cache's index functions (kv4_layout.cuh).
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../llm_fa_b200/csrc/kv4_layout.cuh"

using namespace llmfa;

#define CHECK(c) \
  do { \
    if (!(c)) { \
      std::printf("failed: %s (line %d)\n", #c, __LINE__); \
      std::exit(1); \
    } \
  } while (0)

int main() {
  // both code permutations are permutations, and keep a group's channels in whole words
  bool seen_k[16] = {}, seen_v[32] = {};
  for (int w = 0; w < 16; ++w) seen_k[kv4_key_word(w)] = true;
  for (int w = 0; w < 32; ++w) seen_v[kv4_value_half(w)] = true;
  for (bool s : seen_k) CHECK(s);
  for (bool s : seen_v) CHECK(s);
  for (int ng : {1, 2, 4}) {
    CHECK(kv4_block_bytes(ng) == 2048 + 128 * ng);
    CHECK(kv4_block_bytes(ng) % 128 == 0 && kv4_half_bytes(ng) % 16 == 0);
  }

  for (int shift = 4; shift <= 8; ++shift) {
    std::vector<int32_t> table = {2, -1, 0, 3, /* next row */ 1, 7, 4, 2};
    int32_t lengths[2] = {0, 0};
    int status = 0;
    const Kv4Pool pool{nullptr, nullptr, nullptr, 5, 3, shift, 2};
    const Kv4Seqs seqs{table.data(), 4, 4, 2, lengths, &status};
    const int page = 1 << shift;
    CHECK(kv4_capacity(pool, seqs) == 4 * page);
    CHECK(kv4_page(pool, seqs, 0, 0) == 2 && kv4_page(pool, seqs, 0, page - 1) == 2);
    CHECK(kv4_page(pool, seqs, 0, page) == -1);      // unused entry
    CHECK(kv4_page(pool, seqs, 1, page) == -1);      // id past the pool
    CHECK(kv4_page(pool, seqs, 1, 2 * page) == 4);   // last page of the pool
    CHECK(kv4_page(pool, seqs, 0, 4 * page) == -1);  // past the table
    CHECK(kv4_page(pool, seqs, 0, -1) == -1);
    CHECK(kv4_page(pool, seqs, 1, 1ll << 40) == -1);
    // blocks of a (page, head) are contiguous, pages and heads do not overlap
    std::vector<char> used(5 * 3 * page / 16, 0);
    for (int p = 0; p < 5; ++p)
      for (int h = 0; h < 3; ++h)
        for (int s = 0; s < page; ++s) {
          const long long off = kv4_block_offset(pool, p, h, s + 3 * page);
          CHECK(off % kv4_block_bytes(2) == 0);
          const long long i = off / kv4_block_bytes(2);
          CHECK(i >= 0 && i < static_cast<long long>(used.size()));
          if (s % 16 == 0) CHECK(used[i]++ == 0);
          CHECK(kv4_token_index(pool, p, h, s + page) == (static_cast<long long>(p) * 3 + h) * page + s);
        }
  }
  // offsets past 32 bits
  const Kv4Pool big{nullptr, nullptr, nullptr, 1 << 30, 8, 8, 4};
  CHECK(kv4_block_offset(big, (1 << 30) - 1, 7, 255) ==
        (((1ll << 30) - 1) * 8 + 7) * 16 * 2560 + 15 * 2560);
  CHECK(kv4_token_index(big, (1 << 30) - 1, 7, 255) == (((1ll << 30) - 1) * 8 + 7) * 256 + 255);
  CHECK(kv4_clamp(-1, 5) == 0 && kv4_clamp(6, 5) == 5 && kv4_clamp(3, 5) == 3);
  CHECK(kv4_visible(10, 3, 0, true) == 8 && kv4_visible(10, 3, 2, true) == 10);
  CHECK(kv4_visible(1, 3, 0, true) == 0 && kv4_visible(1, 3, 0, false) == 1);
  std::printf("ok\n");
  return 0;
}
