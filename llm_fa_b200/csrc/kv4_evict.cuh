// Eviction from the 4-bit cache by accumulated attention weight.
//
// select: of a sequence's n slots, n - keep go from every head. They are the
// smallest by weight, then slot; slots whose position is one of the `recent`
// latest are protected: they go after all others, by slot alone. Freed slots below `keep` (holes) and
// surviving slots at or above it (movers) are equally many; the k-th hole takes
// the k-th mover. src[d] is the slot whose token slot d holds afterwards (d
// itself where nothing moves), -1 past the new length.
//
// Measured: 8 sequences of 8192 slots to 4096, 8 heads: 14 us; one of 131,072 to
// 65,536: 27 us (1364 with one CTA a head). Both wait on the chain of passes, not
// on the 8 bytes a slot: cluster barriers take 1 us a digit.
//
// move: carries the tokens out. Sources lie at or above `keep` and targets
// below it, so nothing that is read is written and all moves run at once; a
// cache that stays at its budget moves one token a step, not all of them. Half
// of 64 x 8192 slots: 10 us, 37 MB.
#pragma once
#include "kv4_layout.cuh"
#include "ptx.cuh"

namespace llmfa {

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

// Keys of slots slot .. slot + 3 (slot a multiple of 4: one page holds them).
__device__ __forceinline__ uint4 kv4_slot_keys(const Kv4SelectParams& p, const int32_t* table, int h,
                                               int slot, int n, int first_recent) {
  uint4 k = make_uint4(kKv4Protected, kKv4Protected, kKv4Protected, kKv4Protected);
  if (slot >= n) return k;
  const int page = table[slot >> p.pool.page_shift];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.pool.num_pages)) {
    kv4_report(p.seqs, kStatusKv4BadPage);
    return make_uint4(0, 0, 0, 0);  // slots without a page go first
  }
  const long long i = kv4_token_index(p.pool, page, h, slot);
  const int4 pos = *reinterpret_cast<const int4*>(p.pool.positions + i);
  const float4 w = *reinterpret_cast<const float4*>(p.pool.weights + i);
  k.x = pos.x >= first_recent ? kKv4Protected : kv4_weight_key(w.x);
  k.y = pos.y >= first_recent ? kKv4Protected : kv4_weight_key(w.y);
  k.z = pos.z >= first_recent ? kKv4Protected : kv4_weight_key(w.z);
  k.w = pos.w >= first_recent ? kKv4Protected : kv4_weight_key(w.w);
  return k;
}

// ---------------------------------------------------------------- select
// A cluster of CTAs a (sequence, head), each with an equal run of its slots:
// one SM alone would need a pass over a long cache for every digit.
//
//  1. keys of the run into shared memory (SMEM; a run that does not fit is read
//     again each time), and a histogram of their upper 8 bits;
//  2. every CTA adds up the cluster's histograms and finds the digit of the
//     (n - keep)-th smallest key; the same for the next 8 bits, down to the last;
//  3. a warp walks its rows of 128 slots, 4 a lane, in order: the slots that go
//     are kept as bit masks (of equal keys at the border, those before the last that goes);
//  4. movers are written to a list at their rank, and holes take them from it.
//
// Ranks are ballots within a row, sums over the rows of a warp, over the warps
// of a CTA and over the CTAs of the cluster: six cluster barriers at most.
constexpr int kKv4SelectMaxWarps = 32;
constexpr int kKv4SelectMaxCluster = 8;
constexpr int kKv4SelectKeys = 49152;  // keys that fit a CTA's shared memory (192 KB)
constexpr int kKv4SelectBins = 256;
// A cluster's threads walk src in steps of their number, in 32 bits.
constexpr long long kKv4SelectMaxKeep = (1ll << 31) - kKv4SelectMaxCluster * kKv4SelectMaxWarps * 32;

// Slots of a row for each of a CTA's warps.
__host__ __device__ constexpr int kv4_select_row(int warps) { return 4 * 32 * warps; }

// Slots of one CTA's run: whole rows for whole warps.
__host__ __device__ inline int kv4_select_run(long long n, int ctas, int warps) {
  const long long all = static_cast<long long>(ctas) * kv4_select_row(warps);
  return static_cast<int>((n + all - 1) / all) * kv4_select_row(warps);
}

// CTAs of a cluster; the keys of a run fit in shared memory where that is possible at all.
// Doubled while a CTA has more than 4096 slots and half the SMs would be idle.
__host__ inline int kv4_select_ctas(long long units, long long capacity, int sms) {
  int ctas = 1;
  while (ctas < kKv4SelectMaxCluster &&
         (capacity > static_cast<long long>(ctas) * kKv4SelectKeys ||
          (capacity > static_cast<long long>(ctas) * 4096 && units * ctas * 2 <= 2 * sms)))
    ctas *= 2;
  return ctas;
}
// Warps of a CTA. Few for short runs, and where CTAs are many, as more of them are on an SM then
// and their chains of barriers overlap; many where a CTA has an SM for itself and a long run.
// Measured with 8, 16 and 32 warps, us: 8 x 1000 slots 8, 8, 10; 1664 x 239 24, 45, 88; 512 x 8192
// 33, 37, 49; 64 x 8192 17, 14, 14; 64 x 32,768 29, 25, 33; 8 x 131,072 43, 31, 27; 256 x 32,768
// (one CTA fits an SM) 130, 82, 61. 4 warps win 2 us on less than 256 slots and lose everywhere else.
__host__ inline int kv4_select_warps(long long units, long long capacity, int ctas, int sms) {
  const long long run = (capacity + ctas - 1) / ctas, blocks = units * ctas;
  if (run <= 1024 || (run <= 8192 && blocks > 2 * sms)) return 8;
  return run >= 16384 && (blocks <= sms || run > kKv4SelectKeys / 2) ? kKv4SelectMaxWarps : 16;
}
__host__ __device__ inline bool kv4_select_in_smem(long long capacity) {
  return capacity <= static_cast<long long>(kKv4SelectMaxCluster) * kKv4SelectKeys;
}

__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

struct Kv4SelectSmem {
  alignas(16) uint32_t hist[4][kKv4SelectBins];
  uint32_t found[3];
  uint32_t ties[kKv4SelectMaxWarps];
  uint32_t holes[kKv4SelectMaxWarps], movers[kKv4SelectMaxWarps];
  uint32_t total[2];  // holes and movers of this CTA, for the cluster
};

// The digit of the left-th smallest key: one warp adds up the cluster's
// histograms, 8 bins a lane, and finds the bin that the left-th falls into.
__device__ __forceinline__ void kv4_find_digit(const uint32_t* hist, int ctas, uint32_t prefix,
                                               uint32_t left, uint32_t* found) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = ptx::smem_u32(hist + 8 * lane);
  uint4 v[kKv4SelectMaxCluster][2];
#pragma unroll
  for (int c = 0; c < kKv4SelectMaxCluster; ++c) {
    if (c < ctas) {
      v[c][0] = ld_cluster_v4(ptx::mapa(at, c));
      v[c][1] = ld_cluster_v4(ptx::mapa(at + 16, c));
    } else {
      v[c][0] = v[c][1] = make_uint4(0, 0, 0, 0);
    }
  }
  uint32_t count[8] = {};
#pragma unroll
  for (int c = 0; c < kKv4SelectMaxCluster; ++c)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      count[4 * k] += v[c][k].x;
      count[4 * k + 1] += v[c][k].y;
      count[4 * k + 2] += v[c][k].z;
      count[4 * k + 3] += v[c][k].w;
    }
  uint32_t sum = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += count[k];
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += u;
  }
  uint32_t before = upto - sum;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (before < left && left <= before + count[k]) {
      found[0] = (prefix << 8) | (8 * lane + k);
      found[1] = left - before;
      found[2] = count[k];
    }
    before += count[k];
  }
}

// Exclusive prefix over the warps of one value a warp, for lane 0's use by all its lanes.
template <int WARPS>
__device__ __forceinline__ uint32_t kv4_warps_before(const uint32_t* per_warp, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t v = lane < WARPS ? per_warp[lane] : 0u;
  total = __reduce_add_sync(0xffffffffu, v);
  return __reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
}

// Of 4 ballots, bit `lane` of vote[j] being slot 4 lane + j, how many bits come before this lane's.
__device__ __forceinline__ uint32_t kv4_votes_before(const uint32_t (&vote)[4]) {
  const uint32_t lower = (1u << (threadIdx.x & 31)) - 1u;
  return __popc(vote[0] & lower) + __popc(vote[1] & lower) + __popc(vote[2] & lower) +
         __popc(vote[3] & lower);
}
__device__ __forceinline__ uint32_t kv4_votes(const uint32_t (&vote)[4]) {
  return __popc(vote[0]) + __popc(vote[1]) + __popc(vote[2]) + __popc(vote[3]);
}

template <bool SMEM, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
    kv4_select_kernel(const __grid_constant__ Kv4SelectParams p, int32_t* movers, int ctas) {
  constexpr int kThreads = WARPS * 32;
  extern __shared__ __align__(16) uint8_t select_smem[];
  Kv4SelectSmem& sm = *reinterpret_cast<Kv4SelectSmem*>(select_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = ptx::cluster_ctarank();
  const int bh = blockIdx.x / ctas, h = bh % p.pool.heads, b = bh / p.pool.heads;
  const int n = kv4_length(p.pool, p.seqs, b), go = n - p.keep;
  int32_t* src = p.src + static_cast<long long>(bh) * p.keep;
  if (h == 0 && rank == 0 && threadIdx.x == 0) p.new_lengths[b] = min(n, p.keep);
  if (go <= 0) {  // the whole cluster
    for (int i = rank * kThreads + threadIdx.x; i < p.keep; i += ctas * kThreads)
      src[i] = i < n ? i : -1;
    return;
  }
  movers += static_cast<long long>(bh) * p.keep;
  // positions are int32: a border outside their range protects all or nothing
  const long long border = static_cast<long long>(p.seen != nullptr ? p.seen[b] : n) - p.recent;
  const int first_recent = static_cast<int>(border < INT32_MIN ? INT32_MIN : border);
  const int32_t* table = p.seqs.table + b * p.seqs.table_stride;
  const int run = kv4_select_run(n, ctas, WARPS);
  const int rows = run / kv4_select_row(WARPS);  // of a warp; its rows are consecutive
  const int slot0 = rank * run + (warp * rows) * 128 + 4 * lane;
  uint32_t* masks = reinterpret_cast<uint32_t*>(select_smem + sizeof(Kv4SelectSmem)) + warp * rows * 4;
  uint4* keys = reinterpret_cast<uint4*>(select_smem + sizeof(Kv4SelectSmem) + run / 8) +
                warp * rows * 32 + lane;
  auto keys_at = [&](int r) {  // of row r's four slots of this lane
    return SMEM ? keys[r * 32] : kv4_slot_keys(p, table, h, slot0 + r * 128, n, first_recent);
  };

  for (int i = threadIdx.x; i < 4 * kKv4SelectBins; i += kThreads) (&sm.hist[0][0])[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    const int slot = slot0 + r * 128;
    const uint4 k = kv4_slot_keys(p, table, h, slot, n, first_recent);
    if (SMEM) keys[r * 32] = k;
    const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (slot + j < n) atomicAdd(&sm.hist[0][key[j] >> 24], 1u);
  }
  // Of the keys whose upper bits are `prefix`, `left` of `equals` go. Once all of them do, the
  // lower bits do not matter.
  uint32_t prefix = 0, left = go, equals = n;
  int low = 32;
  uint32_t* hist = sm.hist[0];
#pragma unroll 1
  while (low > 0 && left < equals) {
    if (low < 32) {
#pragma unroll 2
      for (int r = 0; r < rows; ++r) {
        const uint4 k = keys_at(r);
        const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((key[j] >> low) == prefix && slot0 + r * 128 + j < n)
            atomicAdd(&hist[(key[j] >> (low - 8)) & 255u], 1u);
      }
    }
    ptx::cluster_sync();
    if (warp == 0) kv4_find_digit(hist, ctas, prefix, left, sm.found);
    __syncthreads();
    prefix = sm.found[0];
    left = sm.found[1];
    equals = sm.found[2];
    low -= 8;
    hist += kKv4SelectBins;
  }
  // keys up to `last` go; where they do not all, low is 0 and the first `left` equal to it do
  const uint32_t last = (prefix << low) | ((1u << low) - 1u);

  // Where not all equal keys go: those before this CTA, from the last histograms; before this
  // warp, by a walk.
  uint32_t equal = 0;
  if (left < equals) {
    const uint32_t at = ptx::smem_u32(&sm.hist[3][last & 255u]);
    for (uint32_t c = 0; c < rank; ++c) equal += ld_cluster_u32(ptx::mapa(at, c));
    uint32_t mine = 0;
    for (int r = 0; r < rows; ++r) {
      const uint4 k = keys_at(r);
      const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        mine += __popc(__ballot_sync(0xffffffffu, key[j] == last && slot0 + r * 128 + j < n));
    }
    if (lane == 0) sm.ties[warp] = mine;
    __syncthreads();
    uint32_t total;
    equal += kv4_warps_before<WARPS>(sm.ties, total);
  }

  uint32_t holes = 0, moves = 0;
#pragma unroll 2
  for (int r = 0; r < rows; ++r) {
    const int slot = slot0 + r * 128;
    const uint4 k = keys_at(r);
    const uint32_t key[4] = {k.x, k.y, k.z, k.w};
    bool goes[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) goes[j] = slot + j < n && key[j] <= last;
    if (left < equals) {
      uint32_t tie[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) tie[j] = __ballot_sync(0xffffffffu, slot + j < n && key[j] == last);
      uint32_t before = equal + kv4_votes_before(tie);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (slot + j < n && key[j] == last) goes[j] = before++ < left;
      equal += kv4_votes(tie);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t out = __ballot_sync(0xffffffffu, goes[j]);
      const uint32_t low_out = __ballot_sync(0xffffffffu, goes[j] && slot + j < p.keep);
      const uint32_t mover = __ballot_sync(0xffffffffu, !goes[j] && slot + j < n && slot + j >= p.keep);
      holes += __popc(low_out);
      moves += __popc(mover);
      if (lane == 0) masks[r * 4 + j] = out;
    }
  }
  if (lane == 0) {
    sm.holes[warp] = holes;
    sm.movers[warp] = moves;
  }
  __syncthreads();
  uint32_t all_holes, all_moves;
  uint32_t hole = kv4_warps_before<WARPS>(sm.holes, all_holes), move = kv4_warps_before<WARPS>(sm.movers, all_moves);
  if (threadIdx.x == 0) {
    sm.total[0] = all_holes;
    sm.total[1] = all_moves;
  }
  ptx::cluster_sync();
#pragma unroll
  for (uint32_t c = 0; c + 1 < kKv4SelectMaxCluster; ++c) {
    if (c < rank) {
      hole += ld_cluster_u32(ptx::mapa(ptx::smem_u32(&sm.total[0]), c));
      move += ld_cluster_u32(ptx::mapa(ptx::smem_u32(&sm.total[1]), c));
    }
  }
  // The guards on k hold unless the weights change meanwhile, which is the caller's mistake.
  const uint32_t keep = p.keep;
  for (int r = 0; r < rows; ++r) {
    const int slot = slot0 + r * 128;
    if (__all_sync(0xffffffffu, slot + 3 < p.keep || slot >= n)) continue;
    uint32_t vote[4];
    bool mover[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mover[j] = ((masks[r * 4 + j] >> lane) & 1u) == 0 && slot + j < n && slot + j >= p.keep;
      vote[j] = __ballot_sync(0xffffffffu, mover[j]);
    }
    uint32_t k = move + kv4_votes_before(vote);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (mover[j]) {
        if (k < keep) movers[k] = slot + j;
        ++k;
      }
    }
    move += kv4_votes(vote);
  }
  __threadfence();
  ptx::cluster_sync();  // the list is complete; nobody reads another CTA's memory past here
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    const int slot = slot0 + r * 128;
    uint32_t vote[4];
    bool goes[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      goes[j] = ((masks[r * 4 + j] >> lane) & 1u) != 0 && slot + j < p.keep;
      vote[j] = __ballot_sync(0xffffffffu, goes[j]);
    }
    uint32_t k = hole + kv4_votes_before(vote);
    int from[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      from[j] = slot + j;
      if (goes[j]) {
        if (k < keep) from[j] = __ldcg(&movers[k]);
        ++k;
      }
    }
    hole += kv4_votes(vote);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (slot + j < p.keep) src[slot + j] = from[j];
  }
}

// ---------------------------------------------------------------- move
constexpr int kKv4MoveThreads = 256;

struct Kv4MoveParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths unused
  const int32_t* src;
  int keep;
};

template <int NG>
struct Kv4PairWords;
template <>
struct Kv4PairWords<1> {
  using Type = uint32_t;
};
template <>
struct Kv4PairWords<2> {
  using Type = uint2;
};
template <>
struct Kv4PairWords<4> {
  using Type = uint4;
};

// A warp has 32 target slots of one (sequence, head). The lanes whose slot takes
// another token carry its pairs, position and weight, and list where its rows
// lie; then 8 lanes carry a token's two rows of 64 bytes, 16 bytes each.
template <int NG>
__global__ void __launch_bounds__(kKv4MoveThreads)
    kv4_move_kernel(const __grid_constant__ Kv4MoveParams p) {
  __shared__ longlong2 rows[kKv4MoveThreads / 32][32];  // byte offsets: from, to
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int to = (blockIdx.x * kKv4MoveThreads + threadIdx.x);
  const int h = blockIdx.y, b = blockIdx.z;
  const long long unit = static_cast<long long>(b) * p.pool.heads + h;
  const int from = to < p.keep ? p.src[unit * p.keep + to] : -1;
  bool moves = from >= 0 && from != to;
  long long pf = -1, pt = -1;
  if (moves) {
    pf = kv4_page(p.pool, p.seqs, b, from);
    pt = kv4_page(p.pool, p.seqs, b, to);
    if (from < p.keep || pf < 0 || pt < 0) {
      kv4_report(p.seqs, from < p.keep ? kStatusKv4BadSource : kStatusKv4BadPage);
      moves = false;
    }
  }
  const uint32_t vote = __ballot_sync(0xffffffffu, moves);
  if (vote == 0) return;
  if (moves) {
    using Words = typename Kv4PairWords<NG>::Type;
    const long long bf = kv4_block_offset(p.pool, pf, h, from), bt = kv4_block_offset(p.pool, pt, h, to);
    rows[warp][__popc(vote & ((1u << lane) - 1u))] =
        make_longlong2(bf + (from & 15) * kKv4RowBytes, bt + (to & 15) * kKv4RowBytes);
    const long long it = kv4_token_index(p.pool, pt, h, to), jf = kv4_token_index(p.pool, pf, h, from);
    const Words* wf = reinterpret_cast<const Words*>(p.pool.pages + bf + kKv4Block * kKv4RowBytes) + (from & 15);
    Words* wt = reinterpret_cast<Words*>(p.pool.pages + bt + kKv4Block * kKv4RowBytes) + (to & 15);
    constexpr int kSide = kv4_half_bytes(NG) / static_cast<int>(sizeof(Words));
    const Words wk = wf[0], wv = wf[kSide];
    const int32_t position = p.pool.positions[jf];
    const float weight = p.pool.weights[jf];
    wt[0] = wk;
    wt[kSide] = wv;
    p.pool.positions[it] = position;
    p.pool.weights[it] = weight;
  }
  __syncwarp();
  const int n = __popc(vote), part = lane & 7;
  const int at = (part & 3) * 16 + (part >> 2) * kv4_half_bytes(NG);
  for (int i = lane >> 3; i < n; i += 16) {
    uint4 v[4];
    longlong2 r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + 4 * k < n) {
        r[k] = rows[warp][i + 4 * k];
        v[k] = *reinterpret_cast<const uint4*>(p.pool.pages + r[k].x + at);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + 4 * k < n) *reinterpret_cast<uint4*>(p.pool.pages + r[k].y + at) = v[k];
  }
}

}  // namespace llmfa
