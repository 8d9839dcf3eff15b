// Host side of the 4-bit cache's C ABI (include/llm_fa_b200.h): argument
// checks, launch shapes and launches on the caller's stream. No allocation, no
// synchronisation; every check is made before the first CUDA call.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/llm_fa_b200.h"
#include "kv4_attention.cuh"
#include "kv4_evict.cuh"
#include "kv4_quant.cuh"
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
  if (!aligned(c->pages, 16) || !aligned(c->positions, 4) || !aligned(c->weights, 4) ||
      !aligned(s->page_table, 4) || !aligned(s->lengths, 4))
    return LLMFA_ERR_UNSUPPORTED;
  if (c->num_pages >= (int64_t(1) << 31) || c->heads > 1024 || s->batch > kKv4MaxBatch ||
      s->max_pages >= (int64_t(1) << (31 - shift)) || s->table_stride >= (int64_t(1) << 38))
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

int64_t quant_blocks(int64_t rows) {
  return (rows * kKv4RowThreads + kKv4QuantThreads - 1) / kKv4QuantThreads;
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
  const int64_t blocks = quant_blocks(seqs->batch * tokens * cache->heads);
  if (blocks >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.counts = counts;
  p.seen = seen;
  p.tokens = static_cast<int>(tokens);
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto ng) {
    kv4_append_kernel<decltype(t), ng.value>
        <<<static_cast<unsigned>(blocks), kKv4QuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
  const int64_t blocks = quant_blocks(seqs->batch * tokens * cache->heads);
  if (blocks >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.counts = counts;
  p.tokens = static_cast<int>(tokens);
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto ng) {
    kv4_expand_kernel<decltype(t), ng.value>
        <<<static_cast<unsigned>(blocks), kKv4QuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

int llmfa_kv4_attention_workspace_size(int64_t batch, int64_t heads, int64_t heads_q, int64_t tokens,
                                       uint64_t* bytes) {
  if (bytes == nullptr || batch < 1 || heads < 1 || heads_q < 1 || tokens < 1 ||
      heads_q % heads != 0)
    return LLMFA_ERR_INVALID_ARGUMENT;
  if (batch > kKv4MaxBatch || heads_q >= (1 << 24) || tokens >= (1 << 24) ||
      batch * heads_q >= (int64_t(1) << 31) / tokens)
    return LLMFA_ERR_UNSUPPORTED;
  *bytes = static_cast<uint64_t>(batch * heads_q * tokens) * 4;
  return LLMFA_OK;
}

int llmfa_kv4_attention(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs, const void* q,
                        const int64_t q_strides[3], void* o, const int64_t o_strides[3], float* lse,
                        const int64_t lse_strides[2], const int32_t* counts, int64_t heads_q,
                        int64_t tokens, int causal, float softmax_scale, float decay, int dtype,
                        void* workspace, uint64_t workspace_bytes, void* stream) {
  Kv4AttnParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, true, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if ((rc = check_tokens(tokens, dtype, counts)) != LLMFA_OK) return rc;
  if (heads_q < 1 || heads_q % cache->heads != 0) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return LLMFA_ERR_INVALID_ARGUMENT;
  if (decay != decay || decay > 1.f) return LLMFA_ERR_INVALID_ARGUMENT;
  if ((rc = check_rows(q, q_strides, seqs->batch, tokens, heads_q, &p.q)) != LLMFA_OK) return rc;
  if ((rc = check_rows(o, o_strides, seqs->batch, tokens, heads_q, &p.o)) != LLMFA_OK) return rc;
  if (lse != nullptr) {
    if (lse_strides == nullptr || !aligned(lse, 4)) return LLMFA_ERR_INVALID_ARGUMENT;
    if ((seqs->batch > 1 && lse_strides[0] < 1) || (heads_q > 1 && lse_strides[1] < 1))
      return LLMFA_ERR_INVALID_ARGUMENT;
    p.lse_sb = lse_strides[0];
    p.lse_sh = lse_strides[1];
  }
  uint64_t need = 0;
  if ((rc = llmfa_kv4_attention_workspace_size(seqs->batch, cache->heads, heads_q, tokens, &need)) !=
      LLMFA_OK)
    return rc;
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need)
    return LLMFA_ERR_INVALID_ARGUMENT;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  const bool track = decay >= 0.f;
  p.lse = lse;
  p.counts = counts;
  p.row_lse = track ? static_cast<float*>(workspace) : nullptr;
  p.heads_q = static_cast<int>(heads_q);
  p.tokens = static_cast<int>(tokens);
  p.causal = causal != 0;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.decay = decay;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_type_and_groups(dtype, p.pool.ng, [&](auto t, auto) {
    using T = decltype(t);
    kv4_simple_kernel<T><<<static_cast<unsigned>(seqs->batch * heads_q * tokens), kKv4SimpleThreads, 0,
                           st>>>(p);
    if ((rc = launched()) != LLMFA_OK || !track) return rc;
    const dim3 grid(64, static_cast<unsigned>(seqs->batch * cache->heads));
    kv4_simple_weights_kernel<T><<<grid, kKv4SimpleThreads, 0, st>>>(p);
    return launched();
  });
}

int llmfa_kv4_evict_workspace_size(int64_t batch, int64_t heads, int64_t keep, uint64_t* bytes) {
  if (bytes == nullptr || batch < 1 || heads < 1 || keep < 1) return LLMFA_ERR_INVALID_ARGUMENT;
  if (batch > kKv4MaxBatch || heads > 1024 || keep >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
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
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.seen = seen;
  p.src = src;
  p.new_lengths = new_lengths;
  p.keep = static_cast<int>(keep);
  p.recent = static_cast<int>(recent);
  kv4_select_kernel<<<static_cast<unsigned>(seqs->batch * cache->heads), kKv4SelectThreads, 0,
                      static_cast<cudaStream_t>(stream)>>>(p, static_cast<int32_t*>(workspace));
  return launched();
}

int llmfa_kv4_evict_move(const llmfa_kv4_cache* cache, const llmfa_kv4_seqs* seqs,
                         const int32_t* src, int64_t keep, void* stream) {
  Kv4MoveParams p{};
  int rc;
  if ((rc = check_cache(cache, seqs, false, &p.pool, &p.seqs)) != LLMFA_OK) return rc;
  if (src == nullptr || keep < 1) return LLMFA_ERR_INVALID_ARGUMENT;
  if (!aligned(src, 4) || keep >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
  const int64_t blocks =
      (seqs->batch * cache->heads * keep + kKv4MoveThreads - 1) / kKv4MoveThreads;
  if (blocks >= (int64_t(1) << 31)) return LLMFA_ERR_UNSUPPORTED;
  if ((rc = device_status_ptr(&p.seqs.status)) != LLMFA_OK) return rc;
  p.src = src;
  p.keep = static_cast<int>(keep);
  return by_type_and_groups(LLMFA_BF16, p.pool.ng, [&](auto, auto ng) {
    kv4_move_kernel<ng.value><<<static_cast<unsigned>(blocks), kKv4MoveThreads, 0,
                                static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

}  // extern "C"
