// The 4-bit key/value cache: its layout, and the index arithmetic that every
// kernel over it shares. Host code runs the same functions in its tests.
//
// A pool holds pages; a page holds, for every key/value head, page_size / 16
// blocks of 16 tokens. One block is contiguous and a multiple of 128 bytes, so
// that one bulk copy brings keys, values and their scales together:
//
//   key codes    16 tokens x 64 bytes
//   key pairs    16 tokens x NG x 4 bytes    NG = 128 / group (1, 2 or 4)
//   value codes  16 tokens x 64 bytes
//   value pairs  16 tokens x NG x 4 bytes
//
// A pair is (scale, zero), both bf16, scale in the low half: the value of a
// code u in 0..15 is scale * (u - zero), zero an integer in 0..15. Codes are
// unsigned, low bits first.
//
// Within a token's 64 bytes the codes are permuted so that the lane of a warp
// that feeds a matrix instruction finds all of its codes side by side (see
// kv4_attention.cuh):
//   keys    16 words of 8 channels; natural word j * 4 + c is stored at c * 4 + j
//   values  32 half-words of 4 channels; natural half-word k * 8 + g is stored
//           at g * 4 + k
// In both a group of 32, 64 or 128 channels is whole words j (or k), so the
// permutation is the same for every group size.
#pragma once
#include <cstdint>

namespace llmfa {

constexpr int kKv4Dim = 128;        // channels of a head
constexpr int kKv4Block = 16;       // tokens of a block
constexpr int kKv4RowBytes = 64;    // a token's codes, keys or values
constexpr int kKv4MaxBatch = 4096;  // sequences of one call

// Device status words (0 = ok); see llmfa_device_status.
constexpr int kStatusKv4BadPage = 0x2001;    // a page id outside the pool, or no page for a token
constexpr int kStatusKv4BadLength = 0x2002;  // a length or count outside its range
constexpr int kStatusKv4BadSource = 0x2003;  // a move from outside the sequence

__host__ __device__ constexpr int kv4_pair_bytes(int ng) { return kKv4Block * ng * 4; }
__host__ __device__ constexpr int kv4_half_bytes(int ng) {  // keys or values of a block
  return kKv4Block * kKv4RowBytes + kv4_pair_bytes(ng);
}
__host__ __device__ constexpr int kv4_block_bytes(int ng) { return 2 * kv4_half_bytes(ng); }

// Stored position of natural word w (8 channels) of a key row, in words, and of
// natural half-word w (4 channels) of a value row, in half-words.
__host__ __device__ constexpr int kv4_key_word(int w) { return (w & 3) * 4 + (w >> 2); }
__host__ __device__ constexpr int kv4_value_half(int w) { return (w & 7) * 4 + (w >> 3); }

struct Kv4Pool {
  uint8_t* pages;      // [num_pages][heads][page_size / 16 blocks]
  int32_t* positions;  // [num_pages][heads][page_size]
  float* weights;      // [num_pages][heads][page_size]
  long long num_pages;
  int heads;
  int page_shift;  // page_size = 1 << page_shift
  int ng;          // groups of a head
};

struct Kv4Seqs {
  const int32_t* table;  // page ids, table[b * table_stride + i]
  long long table_stride;
  int width;               // page ids of a sequence
  int batch;
  const int32_t* lengths;  // slots of a sequence that hold a token
  int* status;             // device status word
};

__host__ __device__ inline long long kv4_capacity(const Kv4Pool& pool, const Kv4Seqs& seqs) {
  return static_cast<long long>(seqs.width) << pool.page_shift;
}

// Page of `slot` of sequence b, or -1 where the slot is outside the table or
// the id outside the pool: nothing is read or written through it then.
__host__ __device__ inline long long kv4_page(const Kv4Pool& pool, const Kv4Seqs& seqs, int b,
                                              long long slot) {
  if (slot < 0 || slot >= kv4_capacity(pool, seqs)) return -1;
  const long long id = seqs.table[b * seqs.table_stride + (slot >> pool.page_shift)];
  return id >= 0 && id < pool.num_pages ? id : -1;
}

// Byte offset of the block that holds `slot` (of page `page`, head h).
__host__ __device__ inline long long kv4_block_offset(const Kv4Pool& pool, long long page, int h,
                                                      long long slot) {
  const int in_page = static_cast<int>(slot & ((1ll << pool.page_shift) - 1));
  const long long blocks = (page * pool.heads + h) << (pool.page_shift - 4);
  return (blocks + (in_page >> 4)) * kv4_block_bytes(pool.ng);
}

// Index of `slot` in positions and weights.
__host__ __device__ inline long long kv4_token_index(const Kv4Pool& pool, long long page, int h,
                                                     long long slot) {
  return ((page * pool.heads + h) << pool.page_shift) + (slot & ((1ll << pool.page_shift) - 1));
}

// A count read from the device, kept inside [0, most].
__host__ __device__ inline int kv4_clamp(long long n, long long most) {
  return static_cast<int>(n < 0 ? 0 : n > most ? most : n);
}

// Slots that new token i of a sequence sees, of n slots and c new tokens.
__host__ __device__ inline int kv4_visible(int n, int c, int i, bool causal) {
  const int v = causal ? n - (c - 1 - i) : n;
  return v > 0 ? v : 0;
}

#ifdef __CUDACC__
__device__ __forceinline__ void kv4_report(const Kv4Seqs& seqs, int code) {
  atomicCAS(seqs.status, 0, code);
}

// Length of sequence b, inside the table's capacity; one outside is reported.
__device__ __forceinline__ int kv4_length(const Kv4Pool& pool, const Kv4Seqs& seqs, int b) {
  const int n = seqs.lengths[b];
  const long long cap = kv4_capacity(pool, seqs);
  if (n < 0 || n > cap) kv4_report(seqs, kStatusKv4BadLength);
  return kv4_clamp(n, cap);
}
// Count of sequence b, inside [0, tokens]; null counts mean all tokens.
__device__ __forceinline__ int kv4_count(const Kv4Seqs& seqs, const int32_t* counts, int b,
                                         int tokens) {
  if (counts == nullptr) return tokens;
  const int c = counts[b];
  if (c < 0 || c > tokens) kv4_report(seqs, kStatusKv4BadLength);
  return kv4_clamp(c, tokens);
}
#endif

}  // namespace llmfa
