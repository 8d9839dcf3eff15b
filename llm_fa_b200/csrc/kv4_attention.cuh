// Attention of a few new queries over the 4-bit cache: one pass over the
// cache, memory-bound up to some 16 query rows a key head.
//
// For a key head the rows are its new tokens x query heads, in tiles of 8 NT.
// A warp takes 32 tokens at a time:
//
//   S^T[token, row] = K q^T     mma m16n8k16, A = key codes, B = queries
//   x = (S - zero * sum(q)) * scale * row factor      (log2 units, per group)
//   p = 2^(x - m), m the row's running maximum
//   O^T[channel, row] += V^T w,  A = value codes, B = w = p * value scale
//   Z[row] += zero * w          O is O^T - Z at the end
//
// so scales and zeros touch the few scores, never the 128 channels, and the
// rows, not the tokens, are the narrow side of the instruction. tcgen05 would
// pad the rows to 64 or more, and its operands would have to be written out to
// shared memory in 16 bits first, four times the bytes that arrive.
//
// Codes become fp16 by one AND: a nibble u in bits 0-3 is the subnormal u *
// 2^-24, in bits 4-7 u * 2^-20 (mma takes fp16 subnormals exactly); 8 codes
// cost 4 ANDs and a shift. The factor 16 of the odd nibbles is taken out of
// the query fragment for keys, of the output row for values. Products of codes
// with 11-bit numbers are exact in fp32.
//
// Roundings to 16 bits: q is scaled by a power of two per row so that its
// largest element is near 2^13 (bf16 and fp16 values stay exact down to 2^-33
// of it); w is fp16, 11 bits, scaled by a power of two per group so that the
// largest value scale seen so far is in [1/2, 1): the running maximum of the
// softmax, once more, for the scales. Sums, maxima and outputs are fp32.
//
// The row maximum is lazy: p may reach 2^kKv4Slack before O is rescaled, so a
// tile needs one vote instead of a reduction over lanes.
//
// Each warp has its own ring of tiles in shared memory, filled by bulk copies
// (a block of 16 tokens is contiguous, keys and values with their pairs): a
// lane issues them, the warp waits on its own barrier, and warps meet only
// where a unit ends and their parts are joined.
#pragma once
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
  float* part_o;   // workspace: [2 * ctas][8 NT][128], fp32
  float2* part_ml; // [2 * ctas][8 NT]: maximum (log2 units) and sum
  int2* unit;      // [units]: first CTA of a unit, and how many
  float* row_lse;  // [batch][tokens][heads_q], log2 units; null without tracking
  int heads_q, tokens, causal;
  int group, row_tiles;
  int ctas;
  float scale_log2;  // softmax_scale * log2(e)
  float decay;       // weights = decay * weights + sums
  unsigned long long timeout_ns;
};

constexpr int kKv4TokenBlocks = kKv4TileTokens / kKv4Block;  // blocks of a tile
constexpr float kKv4Slack = 6.f;
constexpr int kKv4WeightBits = 8;  // w < 2^(kKv4WeightBits + kKv4Slack)
constexpr int kStatusTimeout = 0x1000;  // + wait site: a bounded wait gave up
constexpr int kSiteKv4Tile = 13;
constexpr unsigned long long kKv4DrainNs = 1000000;
constexpr uint32_t kNibbleLo = 0x000f000fu, kNibbleHi = 0x00f000f0u;

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
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

// What a segment needs of its query rows, in shared memory.
template <int NT, int NG>
struct Kv4Queries {
  uint2 frag[8][NT][32];    // B fragments of the 8 steps of 16 channels
  float sum[NG][8 * NT];    // sum of a group's queries, * 2^-24
  float factor[8 * NT];     // of a score
  int limit[8 * NT];        // slots that the row sees
};

// One warp prepares the 8 rows of n-tile nt. Step 2j has nibbles 0, 4 (b0) and
// 1, 5 (b1) of key word j of the lane, step 2j + 1 nibbles 2, 6 and 3, 7: the
// channels 32 j + 8 c + nibble.
template <typename T, int NT, int NG>
__device__ __forceinline__ void kv4_load_queries(const Kv4AttnParams& p, Kv4Queries<NT, NG>& qs,
                                                 int b, int h, int r0, int n, int c, int nt) {
  const int lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  const Kv4Row row = kv4_row(p, h, c, r0 + 8 * nt + g);
  uint4 raw[4] = {};
  if (row.live) {
    const T* q = static_cast<const T*>(p.q.ptr) + b * p.q.sb + row.i * p.q.st + row.hq * p.q.sh;
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = *reinterpret_cast<const uint4*>(q + 32 * j + 8 * cc);
  }
  float x[4][8], top = 0.f, bad = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&raw[j]);
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
  // 2^e brings the largest element to [2^13, 2^14)
  const int e = min(13 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126);
  const float up = bad == 0.f ? __int_as_float((e + 127) << 23) : 0.f;
  float sum[NG] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float v = (bad == 0.f ? x[j][k] : 0.f) * up * (k & 1 ? 0.0625f : 1.f);
      y[k] = __half2float(__float2half_rn(v));
      sum[j * NG / 4] += y[k] * (k & 1 ? 16.f : 1.f);
    }
    qs.frag[2 * j][nt][lane] = make_uint2(Kv4Type<__half>::pack(y[0], y[4]),
                                          Kv4Type<__half>::pack(y[1], y[5]));
    qs.frag[2 * j + 1][nt][lane] = make_uint2(Kv4Type<__half>::pack(y[2], y[6]),
                                              Kv4Type<__half>::pack(y[3], y[7]));
  }
#pragma unroll
  for (int k = 0; k < NG; ++k) {
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], d);
    if (cc == 0) qs.sum[k][8 * nt + g] = sum[k] * 0x1p-24f;
  }
  if (cc == 0) {
    qs.factor[8 * nt + g] =
        bad == 0.f ? ldexpf(p.scale_log2, 24 - e) : __int_as_float(0x7fc00000);
    qs.limit[8 * nt + g] = row.live ? kv4_visible(n, c, row.i, p.causal) : 0;
  }
}

// ---------------------------------------------------------------- tiles
// A warp's ring of tiles: STAGES buffers of kKv4TokenBlocks blocks, each of
// which holds `BYTES` from the block's start (all of it, or the keys' half).
template <int STAGES, int BYTES>
struct Kv4Ring {
  static constexpr int kTileBytes = kKv4TokenBlocks * BYTES;
  uint32_t base, bars;  // shared addresses
  uint32_t head, tail;  // tiles issued and consumed
  uint32_t have;        // bit 2 * stage + block: that block was copied

  // Copies the blocks of a tile; lane k < kKv4TokenBlocks brings block k, if `src` is not null.
  __device__ __forceinline__ void issue(const uint8_t* src) {
    const int lane = threadIdx.x & 31;
    const uint32_t stage = head % STAGES, bar = bars + stage * 8;
    const uint32_t votes = __ballot_sync(0xffffffffu, lane < kKv4TokenBlocks && src != nullptr);
    have = (have & ~(3u << (2 * stage))) | (votes << (2 * stage));
    if (lane == 0) ptx::mbar_arrive_expect_tx(bar, __popc(votes) * BYTES);
    __syncwarp();
    if (lane < kKv4TokenBlocks && src != nullptr)
      ptx::bulk_load(base + stage * kTileBytes + lane * BYTES, src, BYTES, bar);
    ++head;
  }
  // Waits for the next tile, at most timeout_ns; false when its copies did not arrive (or were
  // not issued, after an earlier one did not).
  __device__ __forceinline__ bool wait(unsigned long long timeout_ns) {
    if (tail == head) return false;
    const uint32_t bar = bars + (tail % STAGES) * 8, parity = (tail / STAGES) & 1;
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = ptx::globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      if (ptx::mbar_try_wait(bar, parity)) return true;
      if ((it & 63u) == 0 && ptx::globaltimer_ns() - t0 > timeout_ns) return false;
    }
  }
  __device__ __forceinline__ uint32_t tile() const { return base + (tail % STAGES) * kTileBytes; }
  __device__ __forceinline__ uint32_t blocks() const { return (have >> (2 * (tail % STAGES))) & 3u; }
  __device__ __forceinline__ void release() {
    __syncwarp();  // every lane has read the tile
    tail += tail != head;
  }
};

// Walks the tiles of a CTA's segments that belong to one warp, ahead of the
// computation, and finds their blocks. Tiles go round the warps.
template <int WARPS>
struct Kv4Loader {
  Kv4Segment seg;
  int tile, n;
  int row_tiles;
  bool more;
  long long page;  // of this lane's block of the tile

  __device__ __forceinline__ void find(const Kv4AttnParams& p, const Kv4Split& s, int warp,
                                       bool fresh) {
    if (fresh && more) {
      tile = seg.lo + warp;
      n = kv4_clamp(p.seqs.lengths[seg.b], kv4_capacity(p.pool, p.seqs));
    }
    while (more && tile >= seg.hi) {
      more = seg.next(s);
      if (more) {
        tile = seg.lo + warp;
        n = kv4_clamp(p.seqs.lengths[seg.b], kv4_capacity(p.pool, p.seqs));
      }
    }
    page = -1;
    const int lane = threadIdx.x & 31;
    const long long slot = static_cast<long long>(tile) * kKv4TileTokens + lane * kKv4Block;
    if (more && lane < kKv4TokenBlocks && slot < n) {
      page = kv4_page(p.pool, p.seqs, seg.b, slot);
      if (page < 0) kv4_report(p.seqs, kStatusKv4BadPage);
    }
  }
  __device__ __forceinline__ void start(const Kv4AttnParams& p, const Kv4Split& s, int cta,
                                        int warp, int tiles_a_head) {
    row_tiles = tiles_a_head;
    more = seg.first(s, cta);
    find(p, s, warp, true);
  }
  template <typename Ring>
  __device__ __forceinline__ void issue(const Kv4AttnParams& p, const Kv4Split& s, Ring& ring,
                                        int warp) {
    if (!more) return;
    const long long slot =
        static_cast<long long>(tile) * kKv4TileTokens + (threadIdx.x & 31) * kKv4Block;
    ring.issue(page >= 0 ? p.pool.pages + kv4_block_offset(p.pool, page, seg.i / row_tiles, slot)
                         : nullptr);
    tile += WARPS;
    find(p, s, warp, false);
  }
};

// Costs of the sequences, summed, into shared memory; every CTA does it alike.
template <int THREADS>
__device__ __forceinline__ void kv4_prefix(const Kv4AttnParams& p, uint32_t* prefix) {
  __shared__ uint32_t warp_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t before = 0;
  if (threadIdx.x == 0) prefix[0] = 0;
  for (int base = 0; base < p.seqs.batch; base += THREADS) {
    const int b = base + threadIdx.x;
    uint32_t v = b < p.seqs.batch ? kv4_tiles(kv4_length(p.pool, p.seqs, b)) + kKv4UnitCost : 0;
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
    if (b < p.seqs.batch) prefix[b + 1] = v + add;
    __syncthreads();
  }
}

// Key codes of 16 tokens times the query rows: the raw scores of tokens a (row
// g of the instruction) and a + 8, then x, in log2 units without the row factor.
template <int NT, int NG, typename Frag>
__device__ __forceinline__ void kv4_scores(uint32_t block, int tok, const uint32_t (&pa)[NG],
                                           const uint32_t (&pb)[NG], const float (&qsum)[NG][NT][2],
                                           Frag frag, float (&x)[NT][4]) {
  const int cc = threadIdx.x & 3;
  const uint4 va = ptx::ld_shared_v4(block + tok * kKv4RowBytes + cc * 16);
  const uint4 vb = ptx::ld_shared_v4(block + (tok + 8) * kKv4RowBytes + cc * 16);
  const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
  float raw[NT][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j % (4 / NG) == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[nt][k] = 0.f;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t ua = wa[j] >> (8 * half), ub = wb[j] >> (8 * half);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint2 f = frag(2 * j + half, nt);
        mma_f16(raw[nt], ua & kNibbleLo, ub & kNibbleLo, ua & kNibbleHi, ub & kNibbleHi, f.x, f.y);
      }
    }
    if ((j + 1) % (4 / NG) == 0) {
      const int grp = j * NG / 4;
      const float2 a = kv4_scale_zero(pa[grp]), b = kv4_scale_zero(pb[grp]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 sz = k < 2 ? a : b;
          const float t = fmaf(-sz.y, qsum[grp][nt][k & 1], raw[nt][k]);
          x[nt][k] = grp == 0 ? t * sz.x : fmaf(t, sz.x, x[nt][k]);
        }
      }
    }
  }
}

// 4 channels of a finished row, and with channel 0 its log-sum-exp.
template <typename T>
__device__ __forceinline__ void kv4_write_row(const Kv4AttnParams& p, int b, int h, int c, int r,
                                              int at, float4 acc, float m, float l) {
  const Kv4Row row = kv4_row(p, h, c, r);
  if (!row.live) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* o = static_cast<T*>(p.o.ptr) + b * p.o.sb + row.i * p.o.st + row.hq * p.o.sh + at;
  *reinterpret_cast<uint2*>(o) = make_uint2(Kv4Type<T>::pack(acc.x * inv, acc.y * inv),
                                            Kv4Type<T>::pack(acc.z * inv, acc.w * inv));
  if (at == 0) {
    const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
    if (p.lse != nullptr) p.lse[b * p.lse_sb + row.hq * p.lse_sh + row.i] = lse2 * 0.69314718055994531f;
    if (p.row_lse != nullptr)
      p.row_lse[(static_cast<long long>(b) * p.tokens + row.i) * p.heads_q + row.hq] = lse2;
  }
}

// ---------------------------------------------------------------- the kernel
template <int NT, int NG, int WARPS, int STAGES>
struct Kv4AttnSmem {
  static constexpr int kJoinBlocks = NT == 1 ? 2 : 1;  // blocks of 32 channels joined at a time
  static constexpr int kJoinRow = 36;                  // floats of a row of 32, free of conflicts
  uint8_t ring[WARPS][STAGES][kKv4TokenBlocks * kv4_block_bytes(NG)];
  float join[WARPS][kJoinBlocks][8 * NT][kJoinRow];
  float2 ml[WARPS][8 * NT];
  Kv4Queries<NT, NG> q;
  uint64_t bar[WARPS][STAGES];
};

template <typename T, int NT, int NG, int WARPS, int STAGES, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
    kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kThreads = WARPS * 32, kRows = 8 * NT;
  using Smem = Kv4AttnSmem<NT, NG, WARPS, STAGES>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem_raw + sizeof(Smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;

  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(ptx::smem_u32(&sm.bar[warp][s]), 1);
    ptx::fence_mbar_init();
  }
  kv4_prefix<kThreads>(p, prefix);
  __syncthreads();
  const Kv4Split split = kv4_split(prefix, p.seqs.batch, p.pool.heads * p.row_tiles, p.ctas);
  const int cta = blockIdx.x;
  if (cta >= split.parts) return;

  Kv4Ring<STAGES, kv4_block_bytes(NG)> ring{ptx::smem_u32(sm.ring[warp]),
                                            ptx::smem_u32(sm.bar[warp]), 0, 0, 0};
  Kv4Loader<WARPS> loader;
  loader.start(p, split, cta, warp, p.row_tiles);
  for (int s = 0; s < STAGES; ++s) loader.issue(p, split, ring, warp);

  // matrix rows g and g + 8 are tokens tok and tok + 8 of a block; columns 2c, 2c + 8 of the
  // values' operand tokens c, c + 8, columns 2c + 1, 2c + 9 tokens c + 4, c + 12
  const int tok = (g >> 1) + 4 * (g & 1);
  unsigned long long limit_ns = p.timeout_ns;

  Kv4Segment seg;
  for (bool more = seg.first(split, cta); more; more = seg.next(split)) {
    const int h = seg.i / p.row_tiles, r0 = (seg.i - h * p.row_tiles) * kRows;
    const int n = kv4_clamp(p.seqs.lengths[seg.b], kv4_capacity(p.pool, p.seqs));
    const int c = kv4_count(p.seqs, p.counts, seg.b, p.tokens);
    if (warp < NT) kv4_load_queries<T, NT, NG>(p, sm.q, seg.b, h, r0, n, c, warp);
    __syncthreads();

    uint2 qf[NT <= 2 ? 8 : 1][NT];
    if constexpr (NT <= 2) {
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) qf[s][nt] = sm.q.frag[s][nt][lane];
    }
    auto frag = [&](int s, int nt) {
      if constexpr (NT <= 2) return qf[s][nt];
      else return sm.q.frag[s][nt][lane];
    };
    float qsum[NG][NT][2], factor[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) qsum[grp][nt][k] = sm.q.sum[grp][8 * nt + 2 * cc + k];
        factor[nt][k] = sm.q.factor[8 * nt + 2 * cc + k];
      }
    // slots below `all` are seen by every live row
    const int all = p.causal ? kv4_visible(n, c, r0 / p.group, true) : n;

    float o[8][NT][4], z[NG][NT][2], m[NT][2], l[NT][2];
    int top[NG];  // exponent of the largest value scale so far, biased
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        m[nt][k] = -INFINITY;
        l[nt][k] = 0.f;
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) z[grp][nt][k] = 0.f;
      }
    }
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) top[grp] = 127 - 100;

    for (int t = seg.lo + warp; t < seg.hi; t += WARPS) {
      uint32_t blocks = ring.blocks();
      if (!ring.wait(limit_ns)) {
        // The copies never came: report, issue no more, give those in flight a moment each.
        kv4_report(p.seqs, kStatusTimeout + kSiteKv4Tile);
        limit_ns = kKv4DrainNs;
        loader.more = false;
        blocks = 0;
      }
      const uint32_t tile = ring.tile();
      const int slot0 = t * kKv4TileTokens;
      // a tile that some row does not see whole: past a limit, or without its blocks
      const bool ragged = slot0 + kKv4TileTokens > all || blocks != 3u;

      float x[2][NT][4];
      uint32_t pv[2][2][NG];  // value pairs of tokens tok and tok + 8 of both blocks
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t block = tile + s * kv4_block_bytes(NG);
        const uint32_t pairs = block + kKv4Block * kKv4RowBytes;
        uint32_t pk[2][NG];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ld_pairs<NG>(pairs + (tok + 8 * u) * 4 * NG, pk[u]);
          ld_pairs<NG>(pairs + kv4_half_bytes(NG) + (tok + 8 * u) * 4 * NG, pv[s][u]);
        }
        kv4_scores<NT, NG>(block, tok, pk[0], pk[1], qsum, frag, x[s]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) x[s][nt][k] *= factor[nt][k & 1];
      }
      uint32_t seen = 0xffffffffu;  // bit (2 s + u) * 2 NT + 2 nt + k
      if (ragged) {
        seen = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int slot = slot0 + 16 * s + tok + 8 * u;
            const bool here = ((blocks >> s) & 1u) != 0;
            bool any = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const bool see = here && slot < sm.q.limit[8 * nt + 2 * cc + k];
                any |= see;
                if (see) seen |= 1u << ((2 * s + u) * 2 * NT + 2 * nt + k);
                else x[s][nt][2 * u + k] = -INFINITY;
              }
            if (!any) {
#pragma unroll
              for (int grp = 0; grp < NG; ++grp) pv[s][u][grp] = 0;
            }
          }
      }

      // maxima and value scales: a vote decides whether anything has to be rescaled
      bool grow = false;
      int ex[NG];
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        ex[grp] = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int e = static_cast<int>((pv[s][u][grp] >> 7) & 255u);
            ex[grp] = max(ex[grp], e == 255 ? 0 : e);
          }
        grow |= ex[grp] > top[grp];
      }
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mx[nt][k] = fmaxf(fmaxf(x[0][nt][k], x[0][nt][2 + k]), fmaxf(x[1][nt][k], x[1][nt][2 + k]));
          grow |= mx[nt][k] > m[nt][k] + kKv4Slack;
        }
      if (__any_sync(0xffffffffu, grow)) {
        float down[NG];
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          const int e = max(top[grp], __reduce_max_sync(0xffffffffu, ex[grp]));
          const int shift = top[grp] - e;  // 2^shift, 0 below fp32's range
          down[grp] = shift < -126 ? 0.f : __int_as_float((shift + 127) << 23);
          top[grp] = e;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float v = mx[nt][k];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
            const float mn = fmaxf(m[nt][k], v);
            const float a = m[nt][k] == -INFINITY ? 1.f : ptx::ex2_mufu(m[nt][k] - mn);
            m[nt][k] = mn;
            l[nt][k] *= a;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) z[grp][nt][k] *= a * down[grp];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[i][nt][k] *= a * down[i * NG / 8];
              o[i][nt][2 + k] *= a * down[i * NG / 8];
            }
          }
      }

#pragma unroll
      for (int s = 0; s < 2; ++s) {
        // p, and w = p * value scale * 2^(weight bits - top), as the product's B operand
        uint32_t wb[NG][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float pr[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float d = x[s][nt][2 * u + k] - m[nt][k];
              pr[k] = ptx::ex2_mufu(d);
              if (ragged && ((seen >> ((2 * s + u) * 2 * NT + 2 * nt + k)) & 1u) == 0) pr[k] = 0.f;
              l[nt][k] += pr[k];
            }
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
              const float2 sz = kv4_scale_zero(pv[s][u][grp]);
              const float f = sz.x * __int_as_float((127 + 127 + kKv4WeightBits - 1 - top[grp]) << 23);
              float w[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                w[k] = pr[k] * f;
                // an unseen token may hold a NaN scale
                if (ragged && ((seen >> ((2 * s + u) * 2 * NT + 2 * nt + k)) & 1u) == 0) w[k] = 0.f;
              }
              const uint32_t h2 = Kv4Type<__half>::pack(w[0], w[1]);
              const float2 back = Kv4Type<__half>::unpack(h2);
              z[grp][nt][0] = fmaf(sz.y, back.x, z[grp][nt][0]);
              z[grp][nt][1] = fmaf(sz.y, back.y, z[grp][nt][1]);
              wb[grp][nt][u] = transpose8x8(h2);
            }
          }
        // value codes of tokens cc, cc + 4, cc + 8, cc + 12: 16 channels a lane
        const uint32_t vals = tile + s * kv4_block_bytes(NG) + kv4_half_bytes(NG) + g * 8;
        uint2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ld_shared_v2(vals + (cc + 4 * i) * kKv4RowBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // channels 32 k + 4 g ..
          const uint32_t sel = (k & 1) ? 0x7632u : 0x5410u;
          const uint32_t ra = k < 2 ? __byte_perm(v[0].x, v[1].x, sel) : __byte_perm(v[0].y, v[1].y, sel);
          const uint32_t rb = k < 2 ? __byte_perm(v[2].x, v[3].x, sel) : __byte_perm(v[2].y, v[3].y, sel);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t ua = ra >> (8 * half), ub = rb >> (8 * half);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t* w = wb[k * NG / 4][nt];
              mma_f16(o[2 * k + half][nt], ua & kNibbleLo, ua & kNibbleHi, ub & kNibbleLo,
                      ub & kNibbleHi, w[0], w[1]);
            }
          }
        }
      }
      ring.release();
      loader.issue(p, split, ring, warp);
    }

    // ---- join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], d);
#pragma unroll
          for (int grp = 0; grp < NG; ++grp)
            z[grp][nt][k] += __shfl_xor_sync(0xffffffffu, z[grp][nt][k], d);
        }
        if (g == 0) sm.ml[warp][8 * nt + 2 * cc + k] = make_float2(m[nt][k], l[nt][k]);
      }
    const Kv4Pieces pieces = kv4_pieces(split, seg.at, seg.tiles);
    const bool whole = pieces.count == 1;
    const int slot = 2 * cta + (seg.lo == 0 ? 1 : 0);
    if (threadIdx.x == 0 && seg.lo == 0)
      p.unit[seg.b * split.hr + seg.i] = make_int2(pieces.first, pieces.count);
    constexpr int kJoin = Smem::kJoinBlocks;
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += kJoin) {
#pragma unroll
      for (int kk = 0; kk < kJoin; ++kk) {
        const int k = k0 + kk, grp = k * NG / 4;
        // 2^24 of the codes, and w's own factor, taken back
        const float back = __int_as_float((top[grp] + 1 - kKv4WeightBits) << 23);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float zz = z[grp][nt][j];
            float4 f;
            f.x = (o[2 * k][nt][j] * 0x1p24f - zz) * back;
            f.y = (o[2 * k][nt][2 + j] * 0x1p20f - zz) * back;
            f.z = (o[2 * k + 1][nt][j] * 0x1p24f - zz) * back;
            f.w = (o[2 * k + 1][nt][2 + j] * 0x1p20f - zz) * back;
            *reinterpret_cast<float4*>(&sm.join[warp][kk][8 * nt + 2 * cc + j][4 * g]) = f;
          }
      }
      __syncthreads();
      // each thread 4 channels of a row, over the warps
      for (int e = threadIdx.x; e < kJoin * kRows * 8; e += kThreads) {
        const int kk = e / (kRows * 8), r = e / 8 % kRows, ch = 4 * (e & 7);
        float top_m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top_m = fmaxf(top_m, sm.ml[w][r].x);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 ml = sm.ml[w][r];
          const float a = ml.x == -INFINITY ? 1.f : ptx::ex2_mufu(ml.x - top_m);
          const float4 f = *reinterpret_cast<const float4*>(&sm.join[w][kk][r][ch]);
          sum = fmaf(a, ml.y, sum);
          acc.x = fmaf(a, f.x, acc.x);
          acc.y = fmaf(a, f.y, acc.y);
          acc.z = fmaf(a, f.z, acc.z);
          acc.w = fmaf(a, f.w, acc.w);
        }
        const int at = 32 * (k0 + kk) + ch;
        if (!whole) {
          *reinterpret_cast<float4*>(p.part_o + (static_cast<long long>(slot) * kRows + r) * kKv4Dim + at) = acc;
          if (at == 0) p.part_ml[static_cast<long long>(slot) * kRows + r] = make_float2(top_m, sum);
        } else {
          kv4_write_row<T>(p, seg.b, h, c, r0 + r, at, acc, top_m, sum);
        }
      }
      __syncthreads();
    }
  }
}

// Joins the pieces of the units that were cut: one block a unit, a thread 4
// channels of a row.
constexpr int kKv4CombineThreads = 256;
template <typename T, int NT>
__global__ void __launch_bounds__(kKv4CombineThreads)
    kv4_combine_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kRows = 8 * NT;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int hr = p.pool.heads * p.row_tiles;
  const int2 unit = p.unit[blockIdx.x];
  if (unit.y == 1) return;
  const int b = blockIdx.x / hr, i = blockIdx.x - b * hr, h = i / p.row_tiles;
  const int r0 = (i - h * p.row_tiles) * kRows;
  const int c = kv4_count(p.seqs, p.counts, b, p.tokens);
#pragma unroll
  for (int e = threadIdx.x; e < kRows * 32; e += kKv4CombineThreads) {
    const int r = e / 32, at = 4 * (e & 31);
    float m = -INFINITY;
    for (int k = 0; k < unit.y; ++k)
      m = fmaxf(m, p.part_ml[static_cast<long long>(kv4_slot(unit.x, k)) * kRows + r].x);
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < unit.y; ++k) {
      const long long row = static_cast<long long>(kv4_slot(unit.x, k)) * kRows + r;
      const float2 ml = p.part_ml[row];
      const float4 f = *reinterpret_cast<const float4*>(p.part_o + row * kKv4Dim + at);
      const float a = ml.x == -INFINITY ? 1.f : ptx::ex2_mufu(ml.x - m);
      l = fmaf(a, ml.y, l);
      acc.x = fmaf(a, f.x, acc.x);
      acc.y = fmaf(a, f.y, acc.y);
      acc.z = fmaf(a, f.z, acc.z);
      acc.w = fmaf(a, f.w, acc.w);
    }
    kv4_write_row<T>(p, b, h, c, r0 + r, at, acc, m, l);
  }
}

// The weight that every cached token received: x again, from the keys' half of
// the cache alone, against the rows' final log-sum-exp. 2^(x - lse) is summed
// over the rows in a fixed order; row tiles past the first add to what the same
// thread wrote.
template <int NT, int NG, int WARPS, int STAGES>
struct Kv4WeightsSmem {
  uint8_t ring[WARPS][STAGES][kKv4TokenBlocks * kv4_half_bytes(NG)];
  Kv4Queries<NT, NG> q;
  float lse[8 * NT];
  int page[WARPS][STAGES][kKv4TokenBlocks];
  uint64_t bar[WARPS][STAGES];
};

template <typename T, int NT, int NG, int WARPS, int STAGES, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
    kv4_weights_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int kThreads = WARPS * 32, kRows = 8 * NT;
  using Smem = Kv4WeightsSmem<NT, NG, WARPS, STAGES>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem_raw + sizeof(Smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(ptx::smem_u32(&sm.bar[warp][s]), 1);
    ptx::fence_mbar_init();
  }
  kv4_prefix<kThreads>(p, prefix);
  __syncthreads();
  const Kv4Split split = kv4_split(prefix, p.seqs.batch, p.pool.heads, gridDim.x);
  const int cta = blockIdx.x;
  if (cta >= split.parts) return;
  Kv4Ring<STAGES, kv4_half_bytes(NG)> ring{ptx::smem_u32(sm.ring[warp]),
                                           ptx::smem_u32(sm.bar[warp]), 0, 0, 0};
  Kv4Loader<WARPS> loader{};
  unsigned long long limit_ns = p.timeout_ns;
  auto issue = [&] {
    if (loader.more && lane < kKv4TokenBlocks)
      sm.page[warp][ring.head % STAGES][lane] = static_cast<int>(loader.page);
    loader.issue(p, split, ring, warp);
  };
  const int tok = (g >> 1) + 4 * (g & 1);
  for (int rt = 0; rt < p.row_tiles; ++rt) {
    loader.start(p, split, cta, warp, 1);
    if (limit_ns != p.timeout_ns) loader.more = false;  // after a timeout
    for (int s = 0; s < STAGES; ++s) issue();
    if (rt == 0) asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows' log-sum-exp
    Kv4Segment seg;
    for (bool more = seg.first(split, cta); more; more = seg.next(split)) {
      const int h = seg.i, r0 = rt * kRows;
      const int n = kv4_clamp(p.seqs.lengths[seg.b], kv4_capacity(p.pool, p.seqs));
      const int c = kv4_count(p.seqs, p.counts, seg.b, p.tokens);
      __syncthreads();  // the last segment's rows are read
      if (warp < NT) kv4_load_queries<T, NT, NG>(p, sm.q, seg.b, h, r0, n, c, warp);
      if (threadIdx.x < kRows) {
        const Kv4Row row = kv4_row(p, h, c, r0 + threadIdx.x);
        sm.lse[threadIdx.x] =
            row.live ? p.row_lse[(static_cast<long long>(seg.b) * p.tokens + row.i) * p.heads_q + row.hq]
                     : INFINITY;
      }
      __syncthreads();
      uint2 qf[NT <= 2 ? 8 : 1][NT];
      if constexpr (NT <= 2) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) qf[s][nt] = sm.q.frag[s][nt][lane];
      }
      auto frag = [&](int s, int nt) {
        if constexpr (NT <= 2) return qf[s][nt];
        else return sm.q.frag[s][nt][lane];
      };
      float qsum[NG][NT][2], factor[NT][2], lse[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = 8 * nt + 2 * cc + k;
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) qsum[grp][nt][k] = sm.q.sum[grp][r];
          factor[nt][k] = sm.q.factor[r];
          lse[nt][k] = sm.lse[r];
        }
      for (int t = seg.lo + warp; t < seg.hi; t += WARPS) {
        uint32_t blocks = ring.blocks();
        if (!ring.wait(limit_ns)) {
          kv4_report(p.seqs, kStatusTimeout + kSiteKv4Tile);
          limit_ns = kKv4DrainNs;
          loader.more = false;
          blocks = 0;
        }
        const uint32_t tile = ring.tile();
        const int slot0 = t * kKv4TileTokens;
        float sum[4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t block = tile + s * kv4_half_bytes(NG);
          uint32_t pk[2][NG];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            ld_pairs<NG>(block + kKv4Block * kKv4RowBytes + (tok + 8 * u) * 4 * NG, pk[u]);
          float x[NT][4];
          kv4_scores<NT, NG>(block, tok, pk[0], pk[1], qsum, frag, x);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int slot = slot0 + 16 * s + tok + 8 * u;
            float w = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float pr = ptx::ex2_mufu(fmaf(x[nt][2 * u + k], factor[nt][k], -lse[nt][k]));
                w += slot < sm.q.limit[8 * nt + 2 * cc + k] ? pr : 0.f;
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
        if (((blocks >> s) & 1u) != 0 && slot < n) {
          const int page = sm.page[warp][ring.tail % STAGES][s];
          float* w = p.pool.weights + kv4_token_index(p.pool, page, h, slot);
          *w = rt > 0 ? *w + mine : p.decay == 0.f ? mine : fmaf(p.decay, *w, mine);
        }
        ring.release();
        issue();
      }
    }
  }
}

}  // namespace llmfa
