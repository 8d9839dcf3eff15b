// Attention of a few new queries over the 4-bit cache, in one pass over it.
//
// For a key head the rows are its new tokens x query heads, in tiles of 8 NT.
// A warp takes 32 tokens at a time:
//
//   S^T[token, row] = (K - zero) q^T   mma m16n8k16, A = key codes, B = queries
//   x = S * row factor * scale         (log2 units, a sum over the groups)
//   p = 2^(x - m), m the row's running maximum
//   O^T[channel, row] += (V - zero)^T w,   A = value codes, w = p * value scale
//
// so scales touch the few scores, never the 128 channels, and the rows, not
// the tokens, are the narrow side of the instruction. tcgen05 would pad the
// rows to 64 or more and take the codes from shared memory in 16 bits, four
// times the bytes that arrive; e4m3, whose first 16 numbers are evenly spaced
// and so hold a code in a byte, is emulated by two fp16 products in mma.sync.
//
// What bounds it is not the memory but the instructions that make operands of
// codes: some 850 a tile (8 rows, groups of 64; 1050 with groups of 32), the
// values' the most. 60 to 63 % of the issue slots are taken, by 12 warps on an SM
// that wait on one another's fixed latencies; the ALU pipe is half busy, the
// matrix pipe a quarter. With 24 rows (1050 a tile) 8 warps take 41 %, and the
// matrix pipe is 44 % busy.
// Measured: 32 sequences of 3.3k to 8.2k tokens, 8 heads, 8 rows: 74 us, 2.9
// TB/s; one of 131,071 tokens, 8 heads, 4 rows, groups of 32: 61 us, 2.7 TB/s;
// without any arithmetic the copies alone take 44 and 35 us, of which 12 are
// launches, the plan and the first loads. 12 warps on an SM have 168 registers:
// a tile of 8 rows needs a few more (spills of up to 8, 76 and 140 bytes a thread
// for groups of 128, 64 and 32). 14 warps with 144 and 16 with 128 spill more (72 and
// 68 us when 12 took 64), 8 were 10 % slower.
//
// Codes become integers of 16 bits. For fp16 by one LOP3 and one HFMA2 a pair: a
// nibble u in bits 0-3 of a half, or'ed with 0x6400, is 1024 + u, in bits 4-7 it
// is 1024 + 16 u; taking off 1024 + zero (after a multiplication with 1/16 for
// the latter: 64 + zero) leaves u - zero exactly. For bf16 in the same way by
// 0x4300, 128 + u; the upper nibble is shifted down first, as bf16 has 7 bits.
//
// Roundings to 16 bits: none of queries and keys, whose products are exact in
// fp32; both have the queries' type. (bf16 queries made fp16 by a power of two a
// row, 72 instead of 74 us for the batch above, lose channels 2^30 below the
// row's largest, which count where their keys are as much larger.) w is the sum
// of two bf16 numbers, 2^-18 of it off: bf16 has fp32's range, so that a token's
// value scale, whatever weight the token has, takes nothing from the precision of
// another's. (One fp16 number with a common exponent for the scales seen, 64
// instead of 72 us, loses the values of tokens whose scales are 2^24 below that
// of a token of no weight.)
// Sums, maxima and outputs are fp32; outputs are summed in units of 2^-24, so
// that weights up to 2^kKv4Slack of many tokens do not pass fp32's range.
//
// The row maximum is lazy: p may reach 2^kKv4Slack before O is rescaled, so a
// tile needs one vote instead of a reduction over lanes.
//
// A warp is a worker of its own (kv4_plan.cuh): it has a ring of tiles in
// shared memory, filled by bulk copies (a block of 16 tokens is contiguous, keys
// and values with their pairs) that a lane issues and the warp waits for, and
// writes what it has of a unit. Warps of a block share nothing but the plan.
#pragma once
#include <type_traits>

#include "../../include/llm_fa_b200.h"
#include "kv4_plan.cuh"
#include "kv4_quant.cuh"
#include "ptx.cuh"

namespace llmfa {

struct Kv4AttnParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths: slots held, the new tokens' included
  Kv4RowView q, o;  // [batch, tokens, heads_q, 128]
  float* lse;       // lse[b * lse_sb + h * lse_sh + i], or null
  long long lse_sb, lse_sh;
  const int32_t* counts;
  float* part_o;    // workspace: [2 * workers][8 NT][128], fp32
  float2* part_ml;  // [2 * workers][8 NT]: maximum (log2 units) and sum
  int2* unit;       // [units]: first worker of a unit, and how many
  float* row_lse;   // [batch][tokens][heads_q], log2 units; null without tracking
  uint8_t* gave_up; // [workers]: 1 where a worker's wait ran out; null without tracking
  float* scores;    // [batch][heads][capacity][rows], log2 units; null where they are not kept
  int heads_q, tokens, causal;
  int fill;  // LLMFA_KV4_FILL_*: what rows past a count get
  int group, row_tiles;
  int workers;  // of the attention kernel, a multiple of 4
  uint64_t page_stride;  // bytes of a page, all heads
  float scale_log2;  // softmax_scale * log2(e)
  float decay;       // weights = decay * weights + sums
  unsigned long long timeout_ns;
};

constexpr int kKv4TokenBlocks = kKv4TileTokens / kKv4Block;  // blocks of a tile
constexpr float kKv4Slack = 6.f;
constexpr float kKv4Unit = 0x1p-24f;  // of values in sums
constexpr int kStatusTimeout = 0x1000;  // + wait site: a bounded wait gave up
constexpr int kSiteKv4Tile = 13;
constexpr unsigned long long kKv4DrainNs = 1000000;  // for copies in flight after that

// ---------------------------------------------------------------- instructions
template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 matrix of 16-bit elements held one row a lane quad.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// A token's NG pairs.
template <int NG>
__device__ __forceinline__ void ld_pairs(uint32_t addr, uint32_t (&w)[NG]) {
  if constexpr (NG == 1) {
    w[0] = ld_shared_u32(addr);
  } else if constexpr (NG == 2) {
    const uint2 v = ld_shared_v2(addr);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    const uint4 v = ptx::ld_shared_v4(addr);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}

// ---------------------------------------------------------------- codes
// Two halves of 1024 + u (nibble 0 of each half of w), or of 1024 + 16 u (nibble 1).
__device__ __forceinline__ uint32_t nibbles_lo(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t nibbles_hi(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// a / 16 - b
__device__ __forceinline__ uint32_t sixteenth_minus(uint32_t a, uint32_t minus_b) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x2c002c00u), "r"(minus_b));
  return r;
}
// What is taken off the two kinds: 1024 + zero, and -(64 + zero).
struct Kv4Zero {
  uint32_t lo, hi;
};
// Of two tokens' pairs, one in each half. A pair read as fp32 is its zero, an integer, plus less
// than 1/16 (the scale's bits are the low end of the mantissa); adding 2^23 + 0x6400 leaves 0x6400
// + zero, the fp16 number 1024 + zero, in the low half.
__device__ __forceinline__ Kv4Zero kv4_zero(uint32_t pair_a, uint32_t pair_b) {
  const uint32_t a = __float_as_uint(__uint_as_float(pair_a) + 8414208.f);
  const uint32_t b = __float_as_uint(__uint_as_float(pair_b) + 8414208.f);
  Kv4Zero z;
  z.lo = __byte_perm(a, b, 0x5410);
  z.hi = sub_f16x2(0x63806380u, z.lo);  // 960 - (1024 + zero)
  return z;
}
// Two codes less their zeros as bf16: 0x4300 + u is 128 + u, whose low nibble alone lies inside the
// mantissa, and so for the zero, 128 + zero.
__device__ __forceinline__ uint32_t kv4_bf16_pair(uint32_t w, uint32_t zero) {
  uint32_t r, d;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(w));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(r), "r"(zero));
  return d;
}
__device__ __forceinline__ uint32_t kv4_bf16_zero(uint32_t pair_a, uint32_t pair_b) {
  return __byte_perm(__float_as_uint(__uint_as_float(pair_a) + 8405760.f),
                     __float_as_uint(__uint_as_float(pair_b) + 8405760.f), 0x5410);
}
// A token's key codes of a group as operands of the queries' type.
template <typename T>
struct Kv4Keys {  // bf16
  uint32_t zero;
  __device__ __forceinline__ explicit Kv4Keys(uint32_t pair) : zero(kv4_bf16_zero(pair, pair)) {}
  // Nibbles 0, 4 and 1, 5 of a word, or in the second half 2, 6 and 3, 7.
  __device__ __forceinline__ void pairs(uint32_t w, int half, uint32_t& first, uint32_t& second) const {
    first = kv4_bf16_pair(w >> (8 * half), zero);
    second = kv4_bf16_pair(w >> (8 * half + 4), zero);
  }
};
template <>
struct Kv4Keys<__half> {
  Kv4Zero zero;
  __device__ __forceinline__ explicit Kv4Keys(uint32_t pair) : zero(kv4_zero(pair, pair)) {}
  __device__ __forceinline__ void pairs(uint32_t w, int half, uint32_t& first, uint32_t& second) const {
    first = sub_f16x2(nibbles_lo(w >> (8 * half)), zero.lo);
    second = sixteenth_minus(nibbles_hi(w >> (8 * half)), zero.hi);
  }
};
__device__ __forceinline__ float kv4_scale(uint32_t pair) { return __uint_as_float(pair << 16); }

// ---------------------------------------------------------------- query rows
// Row r of a key head is new token r / group, query head r % group.
struct Kv4Row {
  int i, hq;
  bool live;
};
__device__ __forceinline__ Kv4Row kv4_row(const Kv4AttnParams& p, int h, int c, int r) {
  const int i = r / p.group;
  return {i, h * p.group + (r - i * p.group), i < c};
}

// The query rows of a segment, as a lane's B fragments: of n-tile nt, lane (g,
// c) has of row g the channels 32 j + 8 c .. + 7, the codes of its word j. Step
// 2j takes nibbles 0, 4 and 1, 5, step 2j + 1 nibbles 2, 6 and 3, 7. Of rows
// 2c, 2c + 1, whose scores the lane gets, it has the factor, which is taken in before the key
// scales: a product of large keys and small queries stays inside fp32. A factor above 1 or below
// 2^-96 is split into `factor` and one that is taken in afterwards (in shared memory).
template <int NT>
struct Kv4Queries {
  static constexpr bool kInRegisters = NT <= 2;  // else in the warp's shared memory
  uint2 frag[8][kInRegisters ? NT : 1];
  uint2* shared;  // [8][NT][32]
  float factor[NT][2];
  uint32_t limits;  // shared address: slots that each row sees; only tiles at a border read them
  int all;          // slots that every live row sees
  bool split;       // some row's factor is split; the second parts are behind the limits

  __device__ __forceinline__ uint2 operator()(int step, int nt) const {
    if constexpr (kInRegisters) return frag[step][nt];
    else return shared[(step * NT + nt) * 32 + (threadIdx.x & 31)];
  }

  template <typename T>
  __device__ __forceinline__ void fetch(const Kv4AttnParams& p, int b, int h, int r0, int c,
                                        uint4 (&raw)[NT][4]) {
    const int g = (threadIdx.x & 31) >> 2, cc = threadIdx.x & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[nt][j] = make_uint4(0, 0, 0, 0);
      const Kv4Row row = kv4_row(p, h, c, r0 + 8 * nt + g);
      if (row.live) {
        const T* q = static_cast<const T*>(p.q.ptr) + b * p.q.sb + row.i * p.q.st + row.hq * p.q.sh;
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[nt][j] = *reinterpret_cast<const uint4*>(q + 32 * j + 8 * cc);
      }
    }
  }

  template <typename T>
  __device__ __forceinline__ void set(const Kv4AttnParams& p, int h, int r0, int n, int c,
                                      const uint4 (&raw)[NT][4]) {
    const int lane = threadIdx.x & 31, cc = lane & 3;
    __syncwarp();  // the last segment's are read
    for (int r = lane; r < 8 * NT; r += 32) {
      const Kv4Row row = kv4_row(p, h, c, r0 + r);
      st_shared_u32(limits + 4 * r, row.live ? kv4_visible(n, c, row.i, p.causal) : 0);
    }
    bool any_after = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4][8], top = 0.f, bad = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* r = reinterpret_cast<const uint32_t*>(&raw[nt][j]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Kv4Type<T>::unpack(r[k]);
          x[j][2 * k] = f.x;
          x[j][2 * k + 1] = f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          bad += f.x * 0.f + f.y * 0.f;  // NaN for NaN and infinities
        }
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        bad += __shfl_xor_sync(0xffffffffu, bad, d);
      }
      // 2^e keeps sums of products with codes inside fp32 (128 of up to 15 times the largest element),
      // and rows of the smallest numbers in its normal range; fp16 needs neither. A row with an
      // infinity or a NaN is zeros with a NaN factor: it becomes NaN, the others do not.
      const int t = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      const int e = std::is_same<T, __half>::value ? 0 : t > 115 ? 115 - t : t < -60 ? -60 - t : 0;
      const float up = __int_as_float((e + 127) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          y[k] = bad == 0.f ? Kv4Type<T>::pack(x[j][k] * up, x[j][k + 4] * up) : 0u;
        if constexpr (kInRegisters) {
          frag[2 * j][nt] = make_uint2(y[0], y[1]);
          frag[2 * j + 1][nt] = make_uint2(y[2], y[3]);
        } else {
          shared[(2 * j * NT + nt) * 32 + lane] = make_uint2(y[0], y[1]);
          shared[((2 * j + 1) * NT + nt) * 32 + lane] = make_uint2(y[2], y[3]);
        }
      }
      float f = ldexpf(p.scale_log2, -e), after = 1.f;
      if (top == 0.f) {  // a row of zeros, or none: any factor will do
        f = 1.f;
      } else if (f > 0x1p96f) {
        after = ldexpf(p.scale_log2, -e - 32);
        f = 0x1p32f;
      } else if (f > 1.f) {
        after = f;
        f = 1.f;
      } else if (f < 0x1p-96f) {
        after = 0x1p-64f;
        f = ldexpf(p.scale_log2, 64 - e);
      }
      if (bad != 0.f) f = __int_as_float(0x7fc00000);
      any_after |= after != 1.f;
      if (cc == 0) st_shared_u32(limits + 4 * (8 * NT + 8 * nt + (lane >> 2)), __float_as_uint(after));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        factor[nt][k] = __shfl_sync(0xffffffffu, f, (2 * cc + k) * 4);
      }
    }
    split = __any_sync(0xffffffffu, any_after);
    all = p.causal ? kv4_visible(n, c, r0 / p.group, true) : n;
    __syncwarp();
  }
  // Of rows 2c, 2c + 1 of n-tile nt.
  __device__ __forceinline__ int2 limit(int nt) const {
    const uint2 v = ld_shared_v2(limits + (8 * nt + 2 * (threadIdx.x & 3)) * 4);
    return make_int2(v.x, v.y);
  }
  __device__ __forceinline__ float2 after(int nt) const {
    const uint2 v = ld_shared_v2(limits + (8 * NT + 8 * nt + 2 * (threadIdx.x & 3)) * 4);
    return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
  }
};

// ---------------------------------------------------------------- tiles
// A warp's ring of tiles: STAGES buffers of kKv4TokenBlocks blocks, each of
// which holds `BYTES` from the block's start (all of it, or the keys' half). A
// barrier each, and behind these two flags: a wait ran out, a page is missing.
template <int STAGES, int BYTES>
struct Kv4Ring {
  static constexpr int kTileBytes = kKv4TokenBlocks * BYTES;
  uint32_t base, bars;  // shared addresses
  uint32_t put = 0, take = 0;  // stages of the next tile to issue and to consume
  uint32_t pending = 0;        // tiles between them
  uint32_t parity = 0;         // of `take`'s barrier
  uint32_t have = 0;           // two bits a pending tile, the next lowest: its blocks that were copied

  // Copies the blocks of a tile; lane k < kKv4TokenBlocks brings block k, where `here`.
  __device__ __forceinline__ void issue(const uint8_t* src, bool here) {
    const int lane = threadIdx.x & 31;
    const uint32_t bar = bars + put * 8, to = base + put * kTileBytes + lane * BYTES;
    const uint32_t votes = __ballot_sync(0xffffffffu, here);
    if (lane == 0) ptx::mbar_arrive_expect_tx(bar, __popc(votes) * BYTES);
    __syncwarp();
    if (here) ptx::bulk_load(to, src, BYTES, bar);
    have |= votes << (2 * pending);
    ++pending;
    put = put + 1 == STAGES ? 0 : put + 1;
  }
  // Waits for the next tile, at most timeout_ns. A lane that gives up sets the warp's flag and goes
  // on with what the buffer holds: the lanes must not part here, as what follows is the whole
  // warp's. Past the next __syncwarp all see the flag, and issue no more; the end reports it.
  __device__ __forceinline__ void wait(unsigned long long timeout_ns) {
    if (pending == 0) return;
    const uint32_t bar = bars + take * 8;
    if (ptx::mbar_try_wait(bar, parity)) return;
    const uint64_t t0 = ptx::globaltimer_ns();
    const unsigned long long limit_ns = failed() ? kKv4DrainNs : timeout_ns;
    for (uint32_t it = 1;; ++it) {
      if (ptx::mbar_try_wait(bar, parity)) return;
      if ((it & 63u) == 0 && ptx::globaltimer_ns() - t0 > limit_ns) break;
    }
    st_shared_u32(bars + STAGES * 8, 1);
  }
  __device__ __forceinline__ bool failed() const { return ld_shared_u32(bars + STAGES * 8) != 0; }
  __device__ __forceinline__ void no_page() const { st_shared_u32(bars + STAGES * 8 + 4, 1); }
  // At the warp's end: atomics at the tiles would cost registers there.
  __device__ __forceinline__ void report(const Kv4Seqs& seqs) const {
    __syncwarp();
    if (ld_shared_u32(bars + STAGES * 8 + 4) != 0) kv4_report(seqs, kStatusKv4BadPage);
    if (failed()) kv4_report(seqs, kStatusTimeout + kSiteKv4Tile);
  }
  __device__ __forceinline__ uint32_t tile() const { return base + take * kTileBytes; }
  __device__ __forceinline__ uint32_t blocks() const { return have & 3u; }
  __device__ __forceinline__ void release() {
    __syncwarp();  // every lane has read the tile
    if (pending == 0) return;
    --pending;
    have >>= 2;
    if (++take == STAGES) {
      take = 0;
      parity ^= 1u;
    }
  }
};

// What a block knows of the sequences, in shared memory.
struct Kv4Plan {
  Kv4Split split;
  const int32_t* held;  // slots of a sequence
  const int32_t* news;  // its new tokens
};

// Walks the tiles of a warp's segments ahead of the computation and finds their blocks. What is
// needed once a segment stays in shared memory: registers are short.
struct Kv4Loader {
  Kv4Segment* seg;       // this warp's, in shared memory
  const int32_t* table;  // of the segment's sequence
  const uint8_t* pages;  // the head's part of page 0
  int slot, left, n;     // first slot of this lane's block of the tile; tiles left of the segment
  bool more;
  int page;  // of the block, or -1: lanes below kKv4TokenBlocks have one

  __device__ __forceinline__ void enter(const Kv4AttnParams& p, const Kv4Plan& plan,
                                        const Kv4Segment& s, int row_tiles) {
    if ((threadIdx.x & 31) == 0) *seg = s;
    __syncwarp();
    const int lane = threadIdx.x & 31;
    slot = s.lo * kKv4TileTokens + lane * kKv4Block;
    left = s.hi - s.lo;
    n = lane < kKv4TokenBlocks ? plan.held[s.b] : 0;
    table = p.seqs.table + s.b * p.seqs.table_stride;
    pages = p.pool.pages + kv4_block_offset(p.pool, 0, s.i / row_tiles, 0);
  }
  template <typename Ring>
  __device__ __forceinline__ void find(const Kv4AttnParams& p, const Ring& ring) {
    page = -1;
    if (slot < n) {  // n is inside the table
      page = table[slot >> p.pool.page_shift];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.pool.num_pages)) {
        page = -1;
        ring.no_page();
      }
    }
  }
  template <typename Ring>
  __device__ __forceinline__ void start(const Kv4AttnParams& p, const Kv4Plan& plan, const Ring& ring,
                                        const Kv4Segment& s, bool any, int row_tiles) {
    more = any;
    if (!more) return;
    enter(p, plan, s, row_tiles);
    find(p, ring);
  }
  template <int NG, typename Ring>
  __device__ __forceinline__ void issue(const Kv4AttnParams& p, const Kv4Plan& plan, Ring& ring,
                                        int row_tiles) {
    if (!more) return;
    if (ring.failed()) {
      more = false;
      return;
    }
    const int block = (slot & ((1 << p.pool.page_shift) - 1)) >> 4;
    ring.issue(pages + static_cast<uint64_t>(page) * p.page_stride + block * kv4_block_bytes(NG),
               page >= 0);
    slot += kKv4TileTokens;
    if (--left == 0) {
      Kv4Segment s = *seg;
      __syncwarp();
      more = s.next(plan.split);
      if (!more) return;
      enter(p, plan, s, row_tiles);
    }
    find(p, ring);
  }
};

// Bytes of shared memory behind a kernel's own for the plan.
__host__ __device__ constexpr size_t kv4_plan_bytes(int batch) {
  return (3 * static_cast<size_t>(batch) + 1) * sizeof(uint32_t);
}
// Every block makes the plan alike: the sequences' lengths and costs, summed, into shared memory.
template <int THREADS>
__device__ __forceinline__ void kv4_make_plan(const Kv4AttnParams& p, int hr, uint32_t* space,
                                              Kv4Plan& plan) {
  __shared__ uint32_t warp_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, batch = p.seqs.batch;
  uint32_t* prefix = space;
  int32_t* held = reinterpret_cast<int32_t*>(space + batch + 1);
  int32_t* news = held + batch;
  uint32_t before = 0;
  if (threadIdx.x == 0) prefix[0] = 0;
  for (int base = 0; base < batch; base += THREADS) {
    const int b = base + threadIdx.x;
    uint32_t v = 0;
    if (b < batch) {
      const int n = kv4_length(p.pool, p.seqs, b);
      held[b] = n;
      news[b] = kv4_count(p.seqs, p.counts, b, p.tokens);
      v = kv4_tiles(n) + kKv4UnitCost;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    uint32_t add = before;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) add += warp_sum[w];
      before += warp_sum[w];
    }
    if (b < batch) prefix[b + 1] = v + add;
    __syncthreads();
  }
  if (threadIdx.x == 0)
    plan = Kv4Plan{kv4_split(prefix, batch, hr, gridDim.x * (THREADS / 32)), held, news};
  __syncthreads();
}
// Workers next to one another go to different blocks: a small problem uses every SM.
__device__ __forceinline__ int kv4_worker() { return (threadIdx.x >> 5) * gridDim.x + blockIdx.x; }

// Key codes of 16 tokens times the query rows: x of tokens a (row g of the
// instruction) and a + 8, in log2 units.
template <typename T, int NT, int NG>
__device__ __forceinline__ void kv4_scores(uint32_t block, int tok, const Kv4Queries<NT>& q,
                                           float (&x)[NT][4]) {
  const uint32_t row = block + tok * kKv4RowBytes + (threadIdx.x & 3) * 16;
  const uint4 va = ptx::ld_shared_v4(row), vb = ptx::ld_shared_v4(row + 8 * kKv4RowBytes);
  const uint32_t pairs = block + kKv4Block * kKv4RowBytes + tok * 4 * NG;
  uint32_t pa[NG], pb[NG];
  ld_pairs<NG>(pairs, pa);
  ld_pairs<NG>(pairs + 8 * 4 * NG, pb);
  const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
  for (int grp = 0; grp < NG; ++grp) {
    Kv4Keys<T> ka(pa[grp]), kb(pb[grp]);
    float raw[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) raw[nt][k] = 0.f;
#pragma unroll
    for (int j = grp * 4 / NG; j < (grp + 1) * 4 / NG; ++j) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t a0, a1, a2, a3;
        ka.pairs(wa[j], half, a0, a2);
        kb.pairs(wb[j], half, a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint2 f = q(2 * j + half, nt);
          mma_16<T>(raw[nt], a0, a1, a2, a3, f.x, f.y);
        }
      }
    }
    const float sa = kv4_scale(pa[grp]), sb = kv4_scale(pb[grp]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float sc = k < 2 ? sa : sb, y = raw[nt][k] * q.factor[nt][k & 1];
        x[nt][k] = grp == 0 ? y * sc : fmaf(y, sc, x[nt][k]);
      }
  }
  if (q.split) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 f = q.after(nt);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[nt][k] *= (k & 1) == 0 ? f.x : f.y;
    }
  }
}

// A warp's running sums over the tokens of a segment.
template <int NT>
struct Kv4State {
  float o[8][NT][4];  // m-tile i: channels 32 (i / 2) + 4 g + 2 (i % 2) and + 1, rows 2c, 2c + 1
  float m[NT][2], l[NT][2];
};

// One tile of 32 tokens. RAGGED: some row does not see all of it (or a block is
// missing): `blocks` says which are here, n what the sequence holds. `scores`,
// if not null, takes the scores of rows r0 .. of the head's `rows`.
template <typename T, int NT, int NG, bool RAGGED>
__device__ __forceinline__ void kv4_tile(Kv4State<NT>& st, uint32_t tile, int tok,
                                         const Kv4Queries<NT>& q, uint32_t blocks, int slot0, int n,
                                         float* scores, int rows, int r0) {
  constexpr int kBlockBytes = kv4_block_bytes(NG);
  const int lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  float x[2][NT][4];
  uint32_t pv[2][2][NG];  // value pairs of tokens tok and tok + 8 of both blocks
  uint32_t seen = 0;      // bit ((2 s + u) * NT + nt) * 2 + k
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t block = tile + s * kBlockBytes;
    kv4_scores<T, NT, NG>(block, tok, q, x[s]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      ld_pairs<NG>(block + kv4_half_bytes(NG) + kKv4Block * kKv4RowBytes + (tok + 8 * u) * 4 * NG,
                   pv[s][u]);
    if constexpr (RAGGED) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int slot = slot0 + 16 * s + tok + 8 * u;
        const bool here = ((blocks >> s) & 1u) != 0;
        if (!here || slot >= n) {
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) pv[s][u][grp] = 0;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int2 limit = q.limit(nt);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (here && slot < (k == 0 ? limit.x : limit.y)) seen |= 1u << (((2 * s + u) * NT + nt) * 2 + k);
            else x[s][nt][2 * u + k] = -INFINITY;
          }
        }
      }
    }
  }

  if (scores != nullptr) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int slot = slot0 + 16 * s + tok + 8 * u;
        if (slot >= n) continue;
        float* to = scores + static_cast<long long>(slot) * rows;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int r = r0 + 8 * nt + 2 * cc + k;
            if (r < rows) to[r] = x[s][nt][2 * u + k];
          }
      }
  }

  // maxima: a vote decides whether anything has to be rescaled
  bool grow = false;
  float mx[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mx[nt][k] = fmaxf(fmaxf(x[0][nt][k], x[0][nt][2 + k]), fmaxf(x[1][nt][k], x[1][nt][2 + k]));
      grow |= mx[nt][k] > st.m[nt][k] + kKv4Slack;
    }
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = mx[nt][k];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
        const float mn = fmaxf(st.m[nt][k], v);
        const float a = st.m[nt][k] == -INFINITY ? 1.f : ptx::ex2_mufu(st.m[nt][k] - mn);
        st.m[nt][k] = mn;
        st.l[nt][k] *= a;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          st.o[i][nt][k] *= a;
          st.o[i][nt][2 + k] *= a;
        }
      }
  }

#pragma unroll
  for (int s = 0; s < 2; ++s) {
    // p, and w = p * value scale in two parts, as the product's B operand
    uint32_t w[NG][NT][2], rest[NG][NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float f[NG];
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) f[grp] = kv4_scale(pv[s][u][grp]) * kKv4Unit;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float pr[2];
        bool see[2] = {true, true};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          pr[k] = ptx::ex2_mufu(x[s][nt][2 * u + k] - st.m[nt][k]);
          if constexpr (RAGGED) {
            see[k] = ((seen >> (((2 * s + u) * NT + nt) * 2 + k)) & 1u) != 0;
            if (!see[k]) pr[k] = 0.f;
          }
          st.l[nt][k] += pr[k];
        }
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          // an unseen token may hold a NaN scale
          const float w0 = see[0] ? pr[0] * f[grp] : 0.f, w1 = see[1] ? pr[1] * f[grp] : 0.f;
          const uint32_t h2 = Kv4Type<__nv_bfloat16>::pack(w0, w1);
          const float2 back = Kv4Type<__nv_bfloat16>::unpack(h2);
          w[grp][nt][u] = transpose8x8(h2);
          rest[grp][nt][u] = transpose8x8(Kv4Type<__nv_bfloat16>::pack(w0 - back.x, w1 - back.y));
        }
      }
    }
    // Columns 2c, 2c + 1 of the values' operand are tokens c, c + 4 of the block, 2c + 8, 2c + 9
    // tokens c + 8, c + 12; a lane holds 16 channels of each, 4 of every 32.
    const uint32_t half = tile + s * kBlockBytes + kv4_half_bytes(NG);
    uint2 v[4];
    uint32_t z[NG][2];
    {
      uint32_t pz[4][NG];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = ld_shared_v2(half + (cc + 4 * i) * kKv4RowBytes + g * 8);
        ld_pairs<NG>(half + kKv4Block * kKv4RowBytes + (cc + 4 * i) * 4 * NG, pz[i]);
        if constexpr (RAGGED) {
          if (((blocks >> s) & 1u) == 0 || slot0 + 16 * s + cc + 4 * i >= n) {
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) pz[i][grp] = 0;
          }
        }
      }
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        z[grp][0] = kv4_bf16_zero(pz[0][grp], pz[1][grp]);
        z[grp][1] = kv4_bf16_zero(pz[2][grp], pz[3][grp]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // channels 32 k + 4 g ..
      const int grp = k * NG / 4;
      const uint32_t sel = (k & 1) ? 0x7632u : 0x5410u;
      const uint32_t ra = k < 2 ? __byte_perm(v[0].x, v[1].x, sel) : __byte_perm(v[0].y, v[1].y, sel);
      const uint32_t rb = k < 2 ? __byte_perm(v[2].x, v[3].x, sel) : __byte_perm(v[2].y, v[3].y, sel);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a0 = kv4_bf16_pair(ra >> (8 * h), z[grp][0]);
        const uint32_t a1 = kv4_bf16_pair(ra >> (8 * h + 4), z[grp][0]);
        const uint32_t a2 = kv4_bf16_pair(rb >> (8 * h), z[grp][1]);
        const uint32_t a3 = kv4_bf16_pair(rb >> (8 * h + 4), z[grp][1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16<__nv_bfloat16>(st.o[2 * k + h][nt], a0, a1, a2, a3, w[grp][nt][0], w[grp][nt][1]);
          mma_16<__nv_bfloat16>(st.o[2 * k + h][nt], a0, a1, a2, a3, rest[grp][nt][0], rest[grp][nt][1]);
        }
      }
    }
  }
}

// Channels `at` + 32 k .. + 3 (in units of kKv4Unit) of a finished row, and with channel 0 its log-sum-exp. A row past its
// sequence's count is left alone or filled; what was summed for it means nothing.
template <typename T, int K>
__device__ __forceinline__ void kv4_write_row(const Kv4AttnParams& p, int b, int h, int c, int r,
                                              int at, const float4 (&f)[K], float m, float l) {
  const Kv4Row row = kv4_row(p, h, c, r);
  const int fill = row.i < p.tokens ? p.fill : 0;
  if (row.live || (fill & LLMFA_KV4_FILL_OUT) != 0) {
    const float inv = l == 0.f ? 0.f : 1.f / kKv4Unit / l;
    T* o = static_cast<T*>(p.o.ptr) + b * p.o.sb + row.i * p.o.st + row.hq * p.o.sh + at;
#pragma unroll
    for (int k = 0; k < K; ++k)
      *reinterpret_cast<uint2*>(o + 32 * k) =
          row.live ? make_uint2(Kv4Type<T>::pack(f[k].x * inv, f[k].y * inv),
                                Kv4Type<T>::pack(f[k].z * inv, f[k].w * inv))
                   : make_uint2(0, 0);
  }
  if (at == 0 && (row.live || (fill & LLMFA_KV4_FILL_LSE) != 0)) {
    const float lse2 = !row.live || l == 0.f ? -INFINITY : m + log2f(l);
    if (p.lse != nullptr) p.lse[b * p.lse_sb + row.hq * p.lse_sh + row.i] = lse2 * 0.69314718055994531f;
    if (p.row_lse != nullptr)
      p.row_lse[(static_cast<long long>(b) * p.tokens + row.i) * p.heads_q + row.hq] = lse2;
  }
}
// Joins a partial result (maximum and sum, output) to another.
__device__ __forceinline__ void kv4_join(float& m, float& l, float4& acc, float2 ml, float4 f) {
  const float mn = fmaxf(m, ml.x);
  // a part without a token has sum and output 0, or NaN: added as it is
  const float a = m == -INFINITY ? 1.f : ptx::ex2_mufu(m - mn);
  const float c = ml.x == -INFINITY ? 1.f : ptx::ex2_mufu(ml.x - mn);
  m = mn;
  l = fmaf(l, a, ml.y * c);
  acc.x = fmaf(acc.x, a, f.x * c);
  acc.y = fmaf(acc.y, a, f.y * c);
  acc.z = fmaf(acc.z, a, f.z * c);
  acc.w = fmaf(acc.w, a, f.w * c);
}

// ---------------------------------------------------------------- the kernel
template <int NT, int NG, int WARPS, int STAGES>
struct Kv4AttnSmem {
  uint8_t ring[WARPS][STAGES][kKv4TokenBlocks * kv4_block_bytes(NG)];
  uint2 q[Kv4Queries<NT>::kInRegisters ? 1 : WARPS][8 * NT * 32];
  Kv4Plan plan;
  Kv4Segment seg[WARPS];
  uint64_t bar[WARPS][STAGES + 1];  // and the ring's flags
  uint2 limit[WARPS][2 * 4 * NT];   // and second factors
};

template <typename T, int NT, int NG, int WARPS, int STAGES, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
    kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kThreads = WARPS * 32, kRows = 8 * NT;
  using Smem = Kv4AttnSmem<NT, NG, WARPS, STAGES>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;

  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(ptx::smem_u32(&sm.bar[warp][s]), 1);
    sm.bar[warp][STAGES] = 0;
    ptx::fence_mbar_init();
  }
  kv4_make_plan<kThreads>(p, p.pool.heads * p.row_tiles,
                          reinterpret_cast<uint32_t*>(smem_raw + sizeof(Smem)), sm.plan);
  const Kv4Plan& plan = sm.plan;
  const int worker = kv4_worker();
  Kv4Segment seg;
  bool more = seg.first(plan.split, worker);
  if (!more) {
    if (lane == 0 && p.gave_up != nullptr) p.gave_up[worker] = 0;
    return;
  }

  Kv4Ring<STAGES, kv4_block_bytes(NG)> ring{ptx::smem_u32(sm.ring[warp]),
                                            ptx::smem_u32(sm.bar[warp])};
  Kv4Queries<NT> q;
  q.shared = sm.q[Kv4Queries<NT>::kInRegisters ? 0 : warp];
  q.limits = ptx::smem_u32(sm.limit[warp]);
  uint4 raw[NT][4];
  auto fetch = [&] {
    const int h = seg.i / p.row_tiles;
    q.template fetch<T>(p, seg.b, h, (seg.i - h * p.row_tiles) * kRows, plan.news[seg.b], raw);
  };
  // Early, while the first tiles are looked up, or a segment's results written, where registers
  // allow it.
  constexpr bool kEarly = NT == 1;
  if (kEarly) fetch();
  Kv4Loader loader;
  loader.seg = &sm.seg[warp];
  loader.start(p, plan, ring, seg, more, p.row_tiles);
  for (int s = 0; s < STAGES; ++s) loader.template issue<NG>(p, plan, ring, p.row_tiles);

  // rows g and g + 8 of the keys' operand are tokens tok and tok + 8 of a block
  const int tok = (g >> 1) + 4 * (g & 1);
  while (more) {
    const int h = seg.i / p.row_tiles, r0 = (seg.i - h * p.row_tiles) * kRows;
    const int n = plan.held[seg.b], c = plan.news[seg.b];
    if (!kEarly) fetch();
    q.template set<T>(p, h, r0, n, c, raw);
    Kv4State<NT> st;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) st.o[i][nt][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        st.m[nt][k] = -INFINITY;
        st.l[nt][k] = 0.f;
      }
    }

    const int rows = p.tokens * p.group;
    float* scores = p.scores == nullptr ? nullptr
                    : p.scores + (static_cast<long long>(seg.b) * p.pool.heads + h) *
                                     kv4_capacity(p.pool, p.seqs) * rows;
    for (int t = seg.lo; t < seg.hi; ++t) {
      const uint32_t blocks = ring.blocks();
      ring.wait(p.timeout_ns);
      const int slot0 = t * kKv4TileTokens;
      if (slot0 + kKv4TileTokens > q.all || blocks != 3u)
        kv4_tile<T, NT, NG, true>(st, ring.tile(), tok, q, blocks, slot0, n, scores, rows, r0);
      else
        kv4_tile<T, NT, NG, false>(st, ring.tile(), tok, q, blocks, slot0, n, scores, rows, r0);
      ring.release();
      loader.template issue<NG>(p, plan, ring, p.row_tiles);
    }

    // ---- the warp's piece: the unit's rows, or a slot of the workspace
    const bool whole = seg.whole();
    const int slot = 2 * worker + (seg.lo == 0 ? 1 : 0);
    if (lane == 0 && seg.lo == 0) {
      const Kv4Pieces pieces = whole ? Kv4Pieces{worker, 1} : kv4_pieces(plan.split, seg.at, seg.tiles);
      p.unit[seg.b * plan.split.hr + seg.i] = make_int2(pieces.first, pieces.count);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // row 2c + j: channels 32 k + 4 g .. + 3
        float l = st.l[nt][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int r = 8 * nt + 2 * cc + j;
        float4 f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          f[k] = make_float4(st.o[2 * k][nt][j], st.o[2 * k][nt][2 + j], st.o[2 * k + 1][nt][j],
                             st.o[2 * k + 1][nt][2 + j]);
        if (whole) {
          kv4_write_row<T, 4>(p, seg.b, h, c, r0 + r, 4 * g, f, st.m[nt][j], l);
        } else {
          const long long row = static_cast<long long>(slot) * kRows + r;
          float4* part = reinterpret_cast<float4*>(p.part_o + row * kKv4Dim + 4 * g);
#pragma unroll
          for (int k = 0; k < 4; ++k) part[8 * k] = f[k];
          if (g == 0) p.part_ml[row] = make_float2(st.m[nt][j], l);
        }
      }
    more = seg.next(plan.split);
    if (kEarly && more) fetch();
  }
  ring.report(p.seqs);
  if (lane == 0 && p.gave_up != nullptr) p.gave_up[worker] = ring.failed();
}

// Joins the pieces of the units that were cut: one block a unit and row; a
// warp's lanes have 4 channels each, and the warps take the pieces in turn, 8
// at once: a long sequence alone is cut into hundreds, whose latency would add
// up otherwise.
constexpr int kKv4CombineWarps = 32;  // at most
template <typename T, int NT>
__global__ void __launch_bounds__(kKv4CombineWarps * 32)
    kv4_combine_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kRows = 8 * NT, kAtOnce = 8;
  __shared__ float4 acc_of[kKv4CombineWarps][32];
  __shared__ float2 ml_of[kKv4CombineWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int hr = p.pool.heads * p.row_tiles, u = blockIdx.x / kRows, r = blockIdx.x % kRows;
  const int b = u / hr, i = u - b * hr, h = i / p.row_tiles, r0 = (i - h * p.row_tiles) * kRows;
  if (r0 + r >= p.tokens * p.group) return;  // no such row
  const int c = kv4_count(p.seqs, p.counts, b, p.tokens);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 unit = p.unit[u];
  if (unit.y == 1) return;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = warp; k0 < unit.y; k0 += kAtOnce * warps) {
    float2 ml[kAtOnce];
    float4 f[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int k = k0 + j * warps;
      ml[j] = make_float2(-INFINITY, 0.f);
      f[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < unit.y) {
        const long long row = static_cast<long long>(kv4_slot(unit.x, k)) * kRows + r;
        ml[j] = p.part_ml[row];
        f[j] = *reinterpret_cast<const float4*>(p.part_o + row * kKv4Dim + 4 * lane);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) kv4_join(m, l, acc, ml[j], f[j]);
  }
  acc_of[warp][lane] = acc;
  if (lane == 0) ml_of[warp] = make_float2(m, l);
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < warps; ++w) kv4_join(m, l, acc, ml_of[w], acc_of[w][lane]);
  const float4 f[1] = {acc};
  kv4_write_row<T, 1>(p, b, h, c, r0 + r, 4 * lane, f, m, l);
}

// ---------------------------------------------------------------- tracked weights
// The weight that a cached token received is the sum over the rows of 2^(x -
// lse), once the rows' log-sum-exp is final. Where the scores were kept (4
// bytes a token and row), a thread adds up a token's, in the order of the rows.
// Weights outlast a call and decide evictions: where a wait of the attention ran
// out, and scores and log-sum-exps mean nothing, they stay as they were.
__device__ __forceinline__ bool kv4_gave_up(const Kv4AttnParams& p, int thread, int threads) {
  const uint32_t* flags = reinterpret_cast<const uint32_t*>(p.gave_up);
  uint32_t any = 0;
  for (int i = thread; i < p.workers / 4; i += threads) any |= flags[i];
  return any != 0;  // as far as this thread has looked
}
constexpr int kKv4SumThreads = 256;
constexpr int kKv4SumRows = 8192;  // most rows (their log-sum-exp is in shared memory)
__global__ void __launch_bounds__(kKv4SumThreads)
    kv4_sum_weights_kernel(const __grid_constant__ Kv4AttnParams p) {
  extern __shared__ float lse_of[];  // [rows]
  const int bh = blockIdx.x, b = bh / p.pool.heads, h = bh - b * p.pool.heads;
  const int n = kv4_clamp(p.seqs.lengths[b], kv4_capacity(p.pool, p.seqs));
  const int c = kv4_count(p.seqs, p.counts, b, p.tokens), rows = p.tokens * p.group;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int r = threadIdx.x; r < rows; r += kKv4SumThreads) {
    const Kv4Row row = kv4_row(p, h, c, r);
    lse_of[r] = row.live ? p.row_lse[(static_cast<long long>(b) * p.tokens + row.i) * p.heads_q + row.hq]
                         : INFINITY;
  }
  if (__syncthreads_or(kv4_gave_up(p, threadIdx.x, kKv4SumThreads))) return;
  const long long first = bh * kv4_capacity(p.pool, p.seqs);
  for (int slot = blockIdx.y * kKv4SumThreads + threadIdx.x; slot < n;
       slot += gridDim.y * kKv4SumThreads) {
    const long long page = kv4_page(p.pool, p.seqs, b, slot);
    if (page < 0) continue;  // reported by the attention
    const float* x = p.scores + (first + slot) * rows;
    float sum = 0.f;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      const float pr = ptx::ex2_mufu(x[r] - lse_of[r]);
      // unseen: -inf, and so may the row's lse be; no such row: lse +inf
      sum += x[r] == -INFINITY || lse_of[r] == INFINITY ? 0.f : pr;
    }
    float* w = p.pool.weights + kv4_token_index(p.pool, page, h, slot);
    *w = p.decay == 0.f ? sum : fmaf(p.decay, *w, sum);
  }
}

// Where they would take too much memory, x is worked out again from the keys'
// half of the cache. Row tiles past the first add to what the same lane wrote.
template <int NT, int NG, int WARPS, int STAGES>
struct Kv4WeightsSmem {
  uint8_t ring[WARPS][STAGES][kKv4TokenBlocks * kv4_half_bytes(NG)];
  uint2 q[Kv4Queries<NT>::kInRegisters ? 1 : WARPS][8 * NT * 32];
  int page[WARPS][STAGES][kKv4TokenBlocks];
  Kv4Plan plan;
  Kv4Segment seg[WARPS];
  uint64_t bar[WARPS][STAGES + 1];  // and the ring's flags
  uint2 limit[WARPS][2 * 4 * NT];   // and second factors
};

template <typename T, int NT, int NG, int WARPS, int STAGES, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
    kv4_weights_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kThreads = WARPS * 32, kRows = 8 * NT;
  using Smem = Kv4WeightsSmem<NT, NG, WARPS, STAGES>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(ptx::smem_u32(&sm.bar[warp][s]), 1);
    sm.bar[warp][STAGES] = 0;
    ptx::fence_mbar_init();
  }
  kv4_make_plan<kThreads>(p, p.pool.heads, reinterpret_cast<uint32_t*>(smem_raw + sizeof(Smem)),
                          sm.plan);
  const Kv4Plan& plan = sm.plan;
  Kv4Segment first;
  if (!first.first(plan.split, kv4_worker())) return;
  Kv4Ring<STAGES, kv4_half_bytes(NG)> ring{ptx::smem_u32(sm.ring[warp]),
                                           ptx::smem_u32(sm.bar[warp])};
  Kv4Loader loader{};
  loader.seg = &sm.seg[warp];
  auto issue = [&] {
    if (loader.more && lane < kKv4TokenBlocks) sm.page[warp][ring.put][lane] = loader.page;
    loader.template issue<NG>(p, plan, ring, 1);
  };
  const int tok = (g >> 1) + 4 * (g & 1);
  Kv4Queries<NT> q;
  q.shared = sm.q[Kv4Queries<NT>::kInRegisters ? 0 : warp];
  q.limits = ptx::smem_u32(sm.limit[warp]);
  for (int rt = 0; rt < p.row_tiles; ++rt) {
    loader.start(p, plan, ring, first, !ring.failed(), 1);  // no more after a timeout
    for (int s = 0; s < STAGES; ++s) issue();
    if (rt == 0) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows' log-sum-exp
      if (__any_sync(0xffffffffu, kv4_gave_up(p, lane, 32))) {
        while (ring.pending > 0) {  // no copy may outlive the block
          ring.wait(p.timeout_ns);
          ring.release();
        }
        break;
      }
    }
    Kv4Segment seg = first;
    for (bool more = true; more; more = seg.next(plan.split)) {
      const int h = seg.i, r0 = rt * kRows, n = plan.held[seg.b], c = plan.news[seg.b];
      uint4 raw[NT][4];
      q.template fetch<T>(p, seg.b, h, r0, c, raw);
      q.template set<T>(p, h, r0, n, c, raw);
      float lse[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const Kv4Row row = kv4_row(p, h, c, r0 + 8 * nt + 2 * cc + k);
          lse[nt][k] = row.live ? p.row_lse[(static_cast<long long>(seg.b) * p.tokens + row.i) * p.heads_q + row.hq]
                                : INFINITY;
        }
      for (int t = seg.lo; t < seg.hi; ++t) {
        const uint32_t blocks = ring.blocks();
        ring.wait(p.timeout_ns);
        const uint32_t tile = ring.tile();
        const int slot0 = t * kKv4TileTokens;
        float sum[4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float x[NT][4];
          kv4_scores<T, NT, NG>(tile + s * kv4_half_bytes(NG), tok, q, x);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int slot = slot0 + 16 * s + tok + 8 * u;
            float w = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int2 limit = q.limit(nt);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float pr = ptx::ex2_mufu(x[nt][2 * u + k] - lse[nt][k]);
                w += slot < (k == 0 ? limit.x : limit.y) ? pr : 0.f;
              }
            }
            sum[2 * s + u] = w;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        }
        // lane cc of a quad stores token cc of its four
        const float mine = cc == 0 ? sum[0] : cc == 1 ? sum[1] : cc == 2 ? sum[2] : sum[3];
        const int s = cc >> 1, slot = slot0 + 16 * s + tok + 8 * (cc & 1);
        if (((blocks >> s) & 1u) != 0 && slot < n && !ring.failed()) {
          const int page = sm.page[warp][ring.take][s];
          float* w = p.pool.weights + kv4_token_index(p.pool, page, h, slot);
          *w = rt > 0 ? *w + mine : p.decay == 0.f ? mine : fmaf(p.decay, *w, mine);
        }
        ring.release();
        issue();
      }
    }
  }
  ring.report(p.seqs);
}

}  // namespace llmfa
