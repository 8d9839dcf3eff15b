// Eviction from the 4-bit cache by accumulated attention weight.
//
// select: of a sequence's n slots, n - keep go from every head. They are the
// smallest by (protected, weight, slot), where a slot is protected when its
// position is one of the `recent` latest. Freed slots below `keep` (holes) and
// surviving slots at or above it (movers) are equally many; the k-th hole takes
// the k-th mover. src[d] is the slot whose token slot d holds afterwards (d
// itself where nothing moves), -1 past the new length.
//
// move: carries the tokens out. Sources lie at or above `keep` and targets
// below it, so nothing that is read is written and all moves run at once; a
// cache that stays at its budget moves one token a step, not all of them.
#pragma once
#include "kv4_layout.cuh"

namespace llmfa {

constexpr int kKv4SelectThreads = 1024;
constexpr uint32_t kKv4Protected = 0xffffffffu;

struct Kv4SelectParams {
  Kv4Pool pool;
  Kv4Seqs seqs;
  const int32_t* seen;  // tokens appended so far, or null: the lengths
  int32_t* src;         // [batch][heads][keep]
  int32_t* new_lengths;
  int keep, recent;
};

// A weight as an unsigned number of the same order: -0 = +0, NaN above all.
__device__ __forceinline__ uint32_t kv4_weight_key(float w) {
  if (w != w) return kKv4Protected - 1;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t kv4_slot_key(const Kv4SelectParams& p, int b, int h, int slot,
                                                 long long first_recent) {
  const long long page = kv4_page(p.pool, p.seqs, b, slot);
  if (page < 0) {
    kv4_report(p.seqs, kStatusKv4BadPage);
    return 0;  // a slot without a page goes first
  }
  const long long i = kv4_token_index(p.pool, page, h, slot);
  return p.pool.positions[i] >= first_recent ? kKv4Protected : kv4_weight_key(p.pool.weights[i]);
}

// Exclusive prefix of `flag` over the block, and the block's total.
__device__ __forceinline__ int kv4_block_rank(bool flag, int* warp_sums, int& total) {
  const uint32_t vote = __ballot_sync(0xffffffffu, flag);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();  // warp_sums of the last call are read
  if (lane == 0) warp_sums[warp] = __popc(vote);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kKv4SelectThreads / 32; ++i) {
    const int s = warp_sums[i];
    before += i < warp ? s : 0;
    total += s;
  }
  return before + __popc(vote & ((1u << lane) - 1u));
}

// One block a (sequence, head): a radix select of the (n - keep)-th smallest
// key, 8 bits a pass, then the holes and the movers in order.
__global__ void __launch_bounds__(kKv4SelectThreads) kv4_select_kernel(Kv4SelectParams p,
                                                                       int32_t* movers) {
  __shared__ int hist[256];
  __shared__ int warp_sums[kKv4SelectThreads / 32];
  __shared__ uint32_t found[2];
  const int h = blockIdx.x % p.pool.heads, b = blockIdx.x / p.pool.heads;
  const int n = kv4_length(p.pool, p.seqs, b);
  const int go = n - p.keep;
  int32_t* src = p.src + static_cast<long long>(blockIdx.x) * p.keep;
  if (h == 0 && threadIdx.x == 0) p.new_lengths[b] = min(n, p.keep);
  if (go <= 0) {
    for (int i = threadIdx.x; i < p.keep; i += kKv4SelectThreads) src[i] = i < n ? i : -1;
    return;
  }
  const long long first_recent =
      static_cast<long long>(p.seen != nullptr ? p.seen[b] : n) - p.recent;
  uint32_t prefix = 0;
  int left = go;  // how many of the keys that start with `prefix` go
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kKv4SelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kKv4SelectThreads) {
      const uint32_t key = kv4_slot_key(p, b, h, i, first_recent);
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int sum = 0, d = 0;
      while (d < 255 && sum + hist[d] < left) sum += hist[d++];
      found[0] = (prefix << 8) | d;
      found[1] = left - sum;
    }
    __syncthreads();
    prefix = found[0];
    left = static_cast<int>(found[1]);
  }
  const uint32_t last = prefix;  // keys below it go, and the first `left` equal to it
  int equal = 0, holes = 0, moved = 0;
  movers += static_cast<long long>(blockIdx.x) * p.keep;
  for (int pass = 0; pass < 2; ++pass) {  // the movers, then the holes that take them
    equal = holes = moved = 0;
    for (int base = 0; base < n; base += kKv4SelectThreads) {
      const int i = base + threadIdx.x;
      const uint32_t key = i < n ? kv4_slot_key(p, b, h, i, first_recent) : kKv4Protected;
      int total;
      const int rank = equal + kv4_block_rank(i < n && key == last, warp_sums, total);
      equal += total;
      const bool goes = i < n && (key < last || (key == last && rank < left));
      const bool mover = i < n && !goes && i >= p.keep;
      const int m = moved + kv4_block_rank(mover, warp_sums, total);
      moved += total;
      const int d = holes + kv4_block_rank(goes && i < p.keep, warp_sums, total);
      holes += total;
      if (pass == 0 && mover) movers[m] = i;
      if (pass == 1 && i < p.keep) src[i] = goes ? movers[d] : i;
    }
    __syncthreads();
  }
}

constexpr int kKv4MoveThreads = 256;

struct Kv4MoveParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths unused
  const int32_t* src;
  int keep;
};

// One thread a target slot: copies the token's rows, pairs, position and weight.
template <int NG>
__global__ void __launch_bounds__(kKv4MoveThreads) kv4_move_kernel(Kv4MoveParams p) {
  const long long i = static_cast<long long>(blockIdx.x) * kKv4MoveThreads + threadIdx.x;
  if (i >= static_cast<long long>(p.seqs.batch) * p.pool.heads * p.keep) return;
  const int from = p.src[i], to = static_cast<int>(i % p.keep);
  if (from < 0 || from == to) return;
  const int bh = static_cast<int>(i / p.keep), h = bh % p.pool.heads, b = bh / p.pool.heads;
  const long long pf = kv4_page(p.pool, p.seqs, b, from), pt = kv4_page(p.pool, p.seqs, b, to);
  if (from < p.keep || pf < 0 || pt < 0) {
    kv4_report(p.seqs, from < p.keep ? kStatusKv4BadSource : kStatusKv4BadPage);
    return;
  }
  const uint8_t* f = p.pool.pages + kv4_block_offset(p.pool, pf, h, from);
  uint8_t* t = p.pool.pages + kv4_block_offset(p.pool, pt, h, to);
  for (int side = 0; side < 2; ++side) {
    for (int c = 0; c < 4; ++c)
      reinterpret_cast<uint4*>(t + (to & 15) * kKv4RowBytes)[c] =
          reinterpret_cast<const uint4*>(f + (from & 15) * kKv4RowBytes)[c];
    for (int c = 0; c < NG; ++c)
      reinterpret_cast<uint32_t*>(t + kKv4Block * kKv4RowBytes)[(to & 15) * NG + c] =
          reinterpret_cast<const uint32_t*>(f + kKv4Block * kKv4RowBytes)[(from & 15) * NG + c];
    f += kv4_half_bytes(NG);
    t += kv4_half_bytes(NG);
  }
  const long long it = kv4_token_index(p.pool, pt, h, to), jf = kv4_token_index(p.pool, pf, h, from);
  p.pool.positions[it] = p.pool.positions[jf];
  p.pool.weights[it] = p.pool.weights[jf];
}

}  // namespace llmfa
