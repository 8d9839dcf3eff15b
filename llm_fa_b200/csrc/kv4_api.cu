// Host side of the 4-bit cache's C ABI (include/llm_fa_b200.h): argument
// checks, launch shapes and launches on the caller's stream. No allocation, no
// synchronisation; every check is made before the first CUDA call.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/llm_fa_b200.h"
#include "kv4_attention.cuh"
#include "kv4_evict.cuh"
#include "kv4_quant.cuh"
#include "kv4_views.h"
#include "setup.h"

namespace {

using namespace llmfa;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// The pool and the sequences of a call, checked. `lengths` may be null where the call reads none.
int check_cache(const llmfa_kv4_cache* c, const llmfa_kv4_seqs* s, bool lengths, Kv4Pool* pool,
                Kv4Seqs* seqs) {
  if (c == nullptr || s == nullptr) return LLMFA_ERR_INVALID_ARGUMENT;
  if (c->pages == nullptr || c->positions == nullptr || c->weights == nullptr ||
      s->page_table == nullptr || (lengths && s->lengths == nullptr))
    return LLMFA_ERR_INVALID_ARGUMENT;
  if (c->num_pages < 1 || c->heads < 1 || s->batch < 1 || s->max_pages < 1)
    return LLMFA_ERR_INVALID_ARGUMENT;
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_size) ++shift;
  if ((1 << shift) != c->page_size) return LLMFA_ERR_INVALID_ARGUMENT;
  if (c->group != 32 && c->group != 64 && c->group != 128) return LLMFA_ERR_INVALID_ARGUMENT;
  if (s->batch > 1 && s->table_stride < s->max_pages) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!aligned(c->pages, 16) || !aligned(c->positions, 16) || !aligned(c->weights, 16) ||
      !aligned(s->page_table, 4) || !aligned(s->lengths, 4))
    return LLMFA_ERR_UNSUPPORTED;
  if (c->num_pages >= (int64_t(1) << 31) || c->heads > 1024 || s->batch > kKv4MaxBatch ||
      s->max_pages >= (int64_t(1) << (30 - shift)) || s->table_stride >= (int64_t(1) << 38))
    return LLMFA_ERR_UNSUPPORTED;
  *pool = Kv4Pool{static_cast<uint8_t*>(c->pages), c->positions, c->weights, c->num_pages,
                  c->heads, shift, kKv4Dim / c->group};
  *seqs = Kv4Seqs{s->page_table, static_cast<long long>(s->table_stride),
                  static_cast<int>(s->max_pages), static_cast<int>(s->batch), s->lengths, nullptr};
  return LLMFA_OK;
}

// One [batch, tokens, heads, 128] view of 16-bit values.
int check_rows(const void* ptr, const int64_t* st, int64_t batch, int64_t tokens, int64_t heads,
               Kv4RowView* view) {
  if (ptr == nullptr || st == nullptr) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!aligned(ptr, 16)) return LLMFA_ERR_UNSUPPORTED;
  const int64_t dims[3] = {batch, tokens, heads};
  int64_t use[3];
  for (int i = 0; i < 3; ++i) {
    use[i] = dims[i] == 1 ? 0 : st[i];  // the stride of a size-1 dimension is never used
    if (dims[i] != 1 && (st[i] <= 0 || st[i] % 8 != 0 || st[i] >= (int64_t(1) << 38)))
      return LLMFA_ERR_UNSUPPORTED;
  }
  *view = Kv4RowView{const_cast<void*>(ptr), use[0], use[1], use[2]};
  return LLMFA_OK;
}

// What a kernel writes through `a` neither meets itself nor what it reads or writes through `b`,
// two views of the same shape.
int check_apart(const Kv4RowView& a, const Kv4RowView& b, int64_t batch, int64_t tokens,
                int64_t heads) {
  const auto view = [&](const Kv4RowView& v) {
    return Kv4View{reinterpret_cast<uintptr_t>(v.ptr), {v.sb, v.st, v.sh}, {batch, tokens, heads}};
  };
  const Kv4View out = view(a), other = view(b);
  return Kv4Meeting(out, nullptr).found() || Kv4Meeting(out, &other).found()
             ? LLMFA_ERR_INVALID_ARGUMENT
             : LLMFA_OK;
}

int check_tokens(int64_t tokens, int dtype, const int32_t* counts) {
  if (tokens < 1 || (dtype != LLMFA_BF16 && dtype != LLMFA_FP16)) return LLMFA_ERR_INVALID_ARGUMENT;
  if (tokens >= (int64_t(1) << 24) || !aligned(counts, 4)) return LLMFA_ERR_UNSUPPORTED;
  return LLMFA_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? LLMFA_OK : LLMFA_ERR_LAUNCH; }

// Calls f(type tag, groups) with the call's type and group count as template arguments.
template <typename F>
int by_type_and_groups(int dtype, int ng, F f) {
  auto groups = [&](auto t) {
    if (ng == 1) return f(t, std::integral_constant<int, 1>{});
    if (ng == 2) return f(t, std::integral_constant<int, 2>{});
    return f(t, std::integral_constant<int, 4>{});
  };
  return dtype == LLMFA_BF16 ? groups(__nv_bfloat16{}) : groups(__half{});
}

// Grid of append and expand: a token's heads in x, sequences in y.
int quant_grid(int64_t batch, int64_t tokens, int64_t heads, dim3* grid) {
  if (tokens * heads >= (int64_t(1) << 31) / kKv4RowThreads) return LLMFA_ERR_UNSUPPORTED;
  *grid = dim3(static_cast<unsigned>((tokens * heads * kKv4RowThreads + kKv4QuantThreads - 1) /
                                     kKv4QuantThreads),
               static_cast<unsigned>(batch));
  return LLMFA_OK;
}

// Rows of a key head, cut into tiles of 8 nt. A pass over the cache takes about 2, 3 and 4 parts of
// time for 8, 16 and 24 rows (8 x 8192 tokens, 8 heads: 31, 41 and 52 us), which decides. Tiles of
// 24 rows have 255 registers and spill up to 196 bytes a thread, with groups of 32; tiles of 32
// rows, tried when 24 took 46 us, took 81.
struct AttnShape {
  int64_t batch, heads, heads_q, tokens;
  int nt, row_tiles;
  int64_t units;
};

int attn_shape(int64_t batch, int64_t heads, int64_t heads_q, int64_t tokens, AttnShape* s) {
  if (batch < 1 || heads < 1 || heads_q < 1 || tokens < 1 || heads_q % heads != 0)
    return LLMFA_ERR_INVALID_ARGUMENT;
  if (batch > kKv4MaxBatch || heads_q >= (1 << 24) || tokens >= (1 << 24) ||
      batch * heads_q >= (int64_t(1) << 31) / tokens)
    return LLMFA_ERR_UNSUPPORTED;
  const int64_t rows = tokens * (heads_q / heads);
  int nt = 1;
  auto tiles_of = [&](int n) { return (rows + 8 * n - 1) / (8 * n); };
  for (int n = 2; n <= 3; ++n)
    if (tiles_of(n) * (n + 1) < tiles_of(nt) * (nt + 1)) nt = n;
  const int64_t tiles = tiles_of(nt);
  *s = AttnShape{batch, heads, heads_q, tokens, nt, static_cast<int>(tiles), batch * heads * tiles};
  if (s->units * 8 * nt >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
  return LLMFA_OK;
}

// Blocks of the attention kernel on an SM, and their shape.
template <int WARPS, int STAGES, int CTAS>
struct AttnShapeOnSm {
  static constexpr int kWarps = WARPS, kStages = STAGES, kCtas = CTAS, kWorkers = WARPS * CTAS;
};
template <int NT>
struct AttnConfig;
template <>
struct AttnConfig<1> : AttnShapeOnSm<6, 2, 2> {};
template <>
struct AttnConfig<2> : AttnShapeOnSm<4, 3, 2> {};
template <>
struct AttnConfig<3> : AttnShapeOnSm<4, 2, 2> {};

int attn_workers(int nt, int sms) {
  constexpr int per_sm[] = {AttnConfig<1>::kWorkers, AttnConfig<2>::kWorkers, AttnConfig<3>::kWorkers};
  static_assert(per_sm[0] % 4 == 0 && per_sm[1] % 4 == 0 && per_sm[2] % 4 == 0, "flags read as words");
  return sms * per_sm[nt - 1];
}

struct AttnLayout {  // byte offsets in the workspace; partial outputs come first
  uint64_t ml, unit, gave_up, row_lse, scores, bytes;
};

// Tracking keeps the scores up to this size; past it the keys are read again. Kept, 16 sequences of
// 4097 tokens with 32 heads of one row (8 MB) are tracked in 15 us, read again in 50.
constexpr uint64_t kMostScores = uint64_t(256) << 20;

// The grid uses at most this many SMs (a B200 has 148), so that the workspace's size follows from
// a call's arguments alone.
constexpr int kMaxSms = 160;

// `capacity`: slots of a sequence where the call tracks, else 0.
AttnLayout attn_layout(const AttnShape& s, int64_t capacity) {
  const uint64_t workers = attn_workers(s.nt, kMaxSms), rows = 2 * workers * 8 * s.nt;
  AttnLayout w;
  w.ml = rows * kKv4Dim * sizeof(float);
  w.unit = w.ml + rows * sizeof(float2);
  w.gave_up = w.unit + static_cast<uint64_t>(s.units) * sizeof(int2);
  w.row_lse = w.gave_up + (capacity > 0 ? (workers + 3) / 4 * 4 : 0);
  const uint64_t rows_all = static_cast<uint64_t>(s.batch * s.heads_q * s.tokens);
  w.scores = (w.row_lse + (capacity > 0 ? rows_all * sizeof(float) : 0) + 15) / 16 * 16;
  const bool keep = capacity > 0 && s.tokens * (s.heads_q / s.heads) <= kKv4SumRows &&
                    static_cast<uint64_t>(capacity) <= kMostScores / sizeof(float) / rows_all;
  w.bytes = w.scores + (keep ? rows_all * capacity * sizeof(float) : 0);
  return w;
}

// A launch that may start while the kernel before it ends, and waits for it itself.
template <typename K>
int launch_after(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
                 const Kv4AttnParams& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return LLMFA_ERR_LAUNCH;
  }
  return LLMFA_OK;
}

// The kernel may use `bytes` of shared memory; asked for once a device.
template <auto Kernel>
int allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return LLMFA_ERR_CUDA;
  }
  if (((done.load(std::memory_order_acquire) >> dev) & 1) != 0) return LLMFA_OK;
  if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(bytes)) != cudaSuccess) {
    cudaGetLastError();
    return LLMFA_ERR_CUDA;
  }
  done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  return LLMFA_OK;
}

template <bool SMEM, int WARPS>
int select_launch_as(const Kv4SelectParams& p, unsigned grid, int ctas, size_t smem, size_t most,
                     int32_t* movers, cudaStream_t st) {
  constexpr auto kernel = kv4_select_kernel<SMEM, WARPS>;
  const int rc = allow_smem<kernel>(most);
  if (rc != LLMFA_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p, movers, ctas) != cudaSuccess) {
    cudaGetLastError();
    return LLMFA_ERR_LAUNCH;
  }
  return LLMFA_OK;
}

int select_launch(const Kv4SelectParams& p, long long capacity, int sms, int32_t* movers,
                  cudaStream_t st) {
  const long long units = static_cast<long long>(p.seqs.batch) * p.pool.heads;
  const int ctas = kv4_select_ctas(units, capacity, sms);
  const bool in_smem = kv4_select_in_smem(capacity);
  const int warps = in_smem ? kv4_select_warps(units, capacity, ctas, sms) : kKv4SelectMaxWarps;
  const int run = kv4_select_run(capacity, ctas, warps);
  const size_t smem = sizeof(Kv4SelectSmem) + static_cast<size_t>(run) / 8 +
                      (in_smem ? static_cast<size_t>(run) * 4 : 0);
  constexpr size_t kMost = 227 * 1024;
  if (smem > kMost || units * ctas >= (1ll << 31)) return LLMFA_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(units * ctas);
  if (!in_smem) return select_launch_as<false, kKv4SelectMaxWarps>(p, grid, ctas, smem, kMost, movers, st);
  if (warps == 8) return select_launch_as<true, 8>(p, grid, ctas, smem, kMost, movers, st);
  if (warps == 16) return select_launch_as<true, 16>(p, grid, ctas, smem, kMost, movers, st);
  return select_launch_as<true, kKv4SelectMaxWarps>(p, grid, ctas, smem, kMost, movers, st);
}

template <typename T, int NT, int NG>
int attn_launch(const Kv4AttnParams& p, const AttnShape& shape, int sms, cudaStream_t st) {
  using C = AttnConfig<NT>;
  constexpr auto kernel = kv4_attention_kernel<T, NT, NG, C::kWarps, C::kStages, C::kCtas>;
  using Smem = Kv4AttnSmem<NT, NG, C::kWarps, C::kStages>;
  constexpr size_t kMost = sizeof(Smem) + kv4_plan_bytes(kKv4MaxBatch);
  static_assert(kMost <= 227 * 1024, "shared memory");
  const size_t plan = kv4_plan_bytes(static_cast<int>(shape.batch));
  int rc;
  if ((rc = allow_smem<kernel>(kMost)) != LLMFA_OK) return rc;
  kernel<<<static_cast<unsigned>(sms * C::kCtas), C::kWarps * 32, sizeof(Smem) + plan, st>>>(p);
  if ((rc = launched()) != LLMFA_OK) return rc;
  // about as many pieces a unit as there are workers for it, or tiles of the longest sequence
  const long long tiles = kv4_capacity(p.pool, p.seqs) / kKv4TileTokens + 1;
  const long long pieces = (sms * C::kWorkers + shape.units - 1) / shape.units;
  int warps = 1;
  while (warps < kKv4CombineWarps && 8 * warps < (pieces < tiles ? pieces : tiles)) warps *= 2;
  if ((rc = launch_after(kv4_combine_kernel<T, NT>, static_cast<unsigned>(shape.units * 8 * NT),
                         warps * 32, 0, st, p)) != LLMFA_OK)
    return rc;
  if (p.row_lse == nullptr) return LLMFA_OK;
  if (p.scores != nullptr) {
    // blocks for every SM several times over; each goes on through its head's slots
    const long long capacity = kv4_capacity(p.pool, p.seqs), heads = shape.batch * shape.heads;
    const long long most = (capacity + kKv4SumThreads - 1) / kKv4SumThreads;
    const long long want = (16ll * sms + heads - 1) / heads;
    const dim3 grid(static_cast<unsigned>(heads), static_cast<unsigned>(want < most ? want : most));
    return launch_after(kv4_sum_weights_kernel, grid, kKv4SumThreads,
                        static_cast<size_t>(p.tokens) * p.group * sizeof(float), st, p);
  }
  constexpr auto weights = kv4_weights_kernel<T, NT, NG, 8, 3, 2>;
  using WSmem = Kv4WeightsSmem<NT, NG, 8, 3>;
  constexpr size_t kMostW = sizeof(WSmem) + kv4_plan_bytes(kKv4MaxBatch);
  static_assert(kMostW <= 227 * 1024, "shared memory");
  if ((rc = allow_smem<weights>(kMostW)) != LLMFA_OK) return rc;
  return launch_after(weights, static_cast<unsigned>(2 * sms), 8 * 32, sizeof(WSmem) + plan, st, p);
}

}  // namespace

extern "C" {

int llmfa_kv4_page_bytes(int32_t page_size, int32_t group, uint64_t* bytes) {
  if (bytes == nullptr || page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0 ||
      (group != 32 && group != 64 && group != 128))
    return LLMFA_ERR_INVALID_ARGUMENT;
  *bytes = static_cast<uint64_t>(page_size / kKv4Block) * kv4_block_bytes(kKv4Dim / group);
  return LLMFA_OK;
}

int llmfa_kv4_append(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs, const void* k,
                     const int64_t k_strides[3], const void* v, const int64_t v_strides[3],
                     const int32_t* counts, const int32_t* seen, int64_t tokens, int dtype,
                     void* stream) {
  Kv4AppendParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, true, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if ((rc = check_tokens(tokens, dtype, counts)) != LLMFA_OK) return rc;
  if ((rc = check_rows(k, k_strides, seqs->batch, tokens, cache->heads, &p.k)) != LLMFA_OK) return rc;
  if ((rc = check_rows(v, v_strides, seqs->batch, tokens, cache->heads, &p.v)) != LLMFA_OK) return rc;
  if (!aligned(seen, 4)) return LLMFA_ERR_UNSUPPORTED;
  dim3 grid;
  if ((rc = quant_grid(seqs->batch, tokens, cache->heads, &grid)) != LLMFA_OK) return rc;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.counts = counts;
  p.seen = seen;
  p.tokens = static_cast<int>(tokens);
  p.heads = Kv4Div(static_cast<uint32_t>(cache->heads));
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto ng) {
    kv4_append_kernel<decltype(t), ng.value>
        <<<grid, kKv4QuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

int llmfa_kv4_expand(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs, void* k,
                     const int64_t k_strides[3], void* v, const int64_t v_strides[3],
                     const int32_t* counts, int64_t tokens, int dtype, void* stream) {
  Kv4ExpandParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, true, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if ((rc = check_tokens(tokens, dtype, counts)) != LLMFA_OK) return rc;
  if ((rc = check_rows(k, k_strides, seqs->batch, tokens, cache->heads, &p.k)) != LLMFA_OK) return rc;
  if ((rc = check_rows(v, v_strides, seqs->batch, tokens, cache->heads, &p.v)) != LLMFA_OK) return rc;
  dim3 grid;
  if ((rc = quant_grid(seqs->batch, tokens, cache->heads, &grid)) != LLMFA_OK) return rc;
  if ((rc = check_apart(p.k, p.v, seqs->batch, tokens, cache->heads)) != LLMFA_OK ||
      (rc = check_apart(p.v, p.k, seqs->batch, tokens, cache->heads)) != LLMFA_OK)
    return rc;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.counts = counts;
  p.tokens = static_cast<int>(tokens);
  p.heads = Kv4Div(static_cast<uint32_t>(cache->heads));
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto ng) {
    kv4_expand_kernel<decltype(t), ng.value>
        <<<grid, kKv4QuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

int llmfa_kv4_attention_workspace_size(int64_t batch, int64_t heads, int64_t heads_q, int64_t tokens,
                                       int64_t capacity, uint64_t* bytes) {
  if (bytes == nullptr || capacity < 0) return LLMFA_ERR_INVALID_ARGUMENT;
  if (capacity >= (int64_t(1) << 30)) return LLMFA_ERR_UNSUPPORTED;
  AttnShape shape;
  const int rc = attn_shape(batch, heads, heads_q, tokens, &shape);
  if (rc == LLMFA_OK) *bytes = attn_layout(shape, capacity).bytes;
  return rc;
}

int llmfa_kv4_attention(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs, const void* q,
                        const int64_t q_strides[3], void* o, const int64_t o_strides[3], float* lse,
                        const int64_t lse_strides[2], const int32_t* counts, int64_t heads_q,
                        int64_t tokens, int causal, float softmax_scale, float decay, int fill,
                        int dtype, void* workspace, uint64_t workspace_bytes, void* stream) {
  Kv4AttnParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, true, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if ((rc = check_tokens(tokens, dtype, counts)) != LLMFA_OK) return rc;
  if (heads_q < 1 || heads_q % cache->heads != 0) return LLMFA_ERR_INVALID_ARGUMENT;
  // it is used times log2(e), which has to stay in fp32's range too
  const float scale_log2 = softmax_scale * 1.4426950408889634f;
  if (!(softmax_scale > 0.f) || !std::isfinite(scale_log2)) return LLMFA_ERR_INVALID_ARGUMENT;
  if (decay != decay || decay > 1.f) return LLMFA_ERR_INVALID_ARGUMENT;
  if ((fill & ~(LLMFA_KV4_FILL_OUT | LLMFA_KV4_FILL_LSE)) != 0) return LLMFA_ERR_INVALID_ARGUMENT;
  if ((rc = check_rows(q, q_strides, seqs->batch, tokens, heads_q, &p.q)) != LLMFA_OK) return rc;
  if ((rc = check_rows(o, o_strides, seqs->batch, tokens, heads_q, &p.o)) != LLMFA_OK) return rc;
  if (lse != nullptr) {
    if (lse_strides == nullptr || !aligned(lse, 4)) return LLMFA_ERR_INVALID_ARGUMENT;
    if ((seqs->batch > 1 && lse_strides[0] < 1) || (heads_q > 1 && lse_strides[1] < 1))
      return LLMFA_ERR_INVALID_ARGUMENT;
    p.lse_sb = lse_strides[0];
    p.lse_sh = lse_strides[1];
  }
  AttnShape shape;
  if ((rc = attn_shape(seqs->batch, cache->heads, heads_q, tokens, &shape)) != LLMFA_OK) return rc;
  // the work split keeps 32-bit sums of the sequences' tiles
  const int64_t capacity = seqs->max_pages << p.pool.page_shift;
  if (seqs->batch * (capacity / kKv4TileTokens + 1 + kKv4UnitCost) >= (int64_t(1) << 32))
    return LLMFA_ERR_UNSUPPORTED;
  if (workspace == nullptr || !aligned(workspace, 16)) return LLMFA_ERR_INVALID_ARGUMENT;
  const AttnLayout ws = attn_layout(shape, decay >= 0.f ? capacity : 0);
  if (workspace_bytes < ws.bytes) return LLMFA_ERR_INVALID_ARGUMENT;
  if ((rc = check_apart(p.o, p.q, seqs->batch, tokens, heads_q)) != LLMFA_OK) return rc;
  int sms = 0;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK || (rc = device_sms(&sms)) != LLMFA_OK)
    return rc;
  sms = sms < kMaxSms ? sms : kMaxSms;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(base);
  p.part_ml = reinterpret_cast<float2*>(base + ws.ml);
  p.unit = reinterpret_cast<int2*>(base + ws.unit);
  p.row_lse = decay >= 0.f ? reinterpret_cast<float*>(base + ws.row_lse) : nullptr;
  p.gave_up = decay >= 0.f ? base + ws.gave_up : nullptr;
  p.workers = attn_workers(shape.nt, sms);
  p.scores = ws.bytes > ws.scores ? reinterpret_cast<float*>(base + ws.scores) : nullptr;
  p.lse = lse;
  p.counts = counts;
  p.heads_q = static_cast<int>(heads_q);
  p.tokens = static_cast<int>(tokens);
  p.causal = causal != 0;
  p.fill = fill;
  p.group = static_cast<int>(heads_q / cache->heads);
  p.row_tiles = shape.row_tiles;
  p.page_stride = static_cast<uint64_t>(kv4_block_offset(p.pool, 1, 0, 0));
  p.scale_log2 = scale_log2;
  p.decay = decay;
  p.timeout_ns = wait_limit_ns();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto ng) {
    using T = decltype(t);
    if (shape.nt == 1) return attn_launch<T, 1, ng.value>(p, shape, sms, st);
    if (shape.nt == 2) return attn_launch<T, 2, ng.value>(p, shape, sms, st);
    return attn_launch<T, 3, ng.value>(p, shape, sms, st);
  });
}

int llmfa_kv4_evict_workspace_size(int64_t batch, int64_t heads, int64_t keep, uint64_t* bytes) {
  if (bytes == nullptr || batch < 1 || heads < 1 || keep < 1) return LLMFA_ERR_INVALID_ARGUMENT;
  if (batch > kKv4MaxBatch || heads > 1024 || keep > kKv4SelectMaxKeep) return LLMFA_ERR_UNSUPPORTED;
  *bytes = static_cast<uint64_t>(batch * heads * keep) * 4;
  return LLMFA_OK;
}

int llmfa_kv4_evict_select(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs,
                           const int32_t* seen, int64_t keep, int64_t recent, int32_t* src,
                           int32_t* new_lengths, void* workspace, uint64_t workspace_bytes,
                           void* stream) {
  Kv4SelectParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, true, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if (keep < 1 || recent < 0 || recent > keep || src == nullptr || new_lengths == nullptr)
    return LLMFA_ERR_INVALID_ARGUMENT;
  uint64_t need = 0;
  if ((rc = llmfa_kv4_evict_workspace_size(seqs->batch, cache->heads, keep, &need)) != LLMFA_OK)
    return rc;
  if (workspace == nullptr || workspace_bytes < need) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!aligned(seen, 4) || !aligned(src, 4) || !aligned(new_lengths, 4) || !aligned(workspace, 16))
    return LLMFA_ERR_UNSUPPORTED;
  // one block writes a new length while others read the old one
  const uintptr_t was = reinterpret_cast<uintptr_t>(seqs->lengths);
  const uintptr_t is = reinterpret_cast<uintptr_t>(new_lengths), bytes = 4 * seqs->batch;
  if (was < is + bytes && is < was + bytes) return LLMFA_ERR_INVALID_ARGUMENT;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.seen = seen;
  p.src = src;
  p.new_lengths = new_lengths;
  p.keep = static_cast<int>(keep);
  p.recent = static_cast<int>(recent);
  int sms = 0;
  if ((rc = device_sms(&sms)) != LLMFA_OK) return rc;
  return select_launch(p, kv4_capacity(p.pool, p.seqs), sms, static_cast<int32_t*>(workspace),
                       static_cast<cudaStream_t>(stream));
}

int llmfa_kv4_evict_move(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs,
                         const int32_t* src, int64_t keep, void* stream) {
  Kv4MoveParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, false, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if (src == nullptr || keep < 1) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!aligned(src, 4) || keep > (int64_t(1) << 31) - 1024) return LLMFA_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>((keep + kKv4MoveThreads - 1) / kKv4MoveThreads),
                  static_cast<unsigned>(cache->heads), static_cast<unsigned>(seqs->batch));
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.src = src;
  p.keep = static_cast<int>(keep);
  return by_type_and_groups(LLMFA_BF16, p.pool.ng, [&](auto, auto ng) {
    kv4_move_kernel<ng.value><<<grid, kKv4MoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

}  // extern "C"
