// Attention of a few new queries over the 4-bit cache.
#pragma once
#include "kv4_quant.cuh"

namespace llmfa {

struct Kv4AttnParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths: slots held, the new tokens' included
  Kv4RowView q, o;  // [batch, tokens, heads_q, 128]
  float* lse;       // lse[b * lse_sb + h * lse_sh + i], or null
  long long lse_sb, lse_sh;
  const int32_t* counts;
  float* row_lse;  // workspace [batch][tokens][heads_q], log2 units (tracking only)
  int heads_q, tokens, causal;
  float scale_log2;  // softmax_scale * log2(e)
  float decay;       // weights = decay * weights + sums
};

constexpr int kKv4SimpleThreads = 128;

// One value of a token's row.
__device__ __forceinline__ float kv4_value_at(const uint8_t* half, int ng, int tok, int ch,
                                              bool value) {
  const int byte = value ? kv4_value_half(ch / 4) * 2 + (ch % 4) / 2
                         : kv4_key_word(ch / 8) * 4 + (ch % 8) / 2;
  const int code = (half[tok * kKv4RowBytes + byte] >> (4 * (ch & 1))) & 15;
  const float2 sz = kv4_scale_zero(reinterpret_cast<const uint32_t*>(
      half + kKv4Block * kKv4RowBytes)[tok * ng + ch / (kKv4Dim / ng)]);
  return sz.x * (static_cast<float>(code) - sz.y);
}

// One block a query row; a tile of 128 keys at a time.
template <typename T>
__global__ void __launch_bounds__(kKv4SimpleThreads) kv4_simple_kernel(Kv4AttnParams p) {
  __shared__ float q[kKv4Dim], prob[kKv4SimpleThreads], red[4];
  const int hq = blockIdx.x % p.heads_q, i = blockIdx.x / p.heads_q % p.tokens,
            b = blockIdx.x / p.heads_q / p.tokens, h = hq / (p.heads_q / p.pool.heads);
  const int n = kv4_length(p.pool, p.seqs, b), c = kv4_count(p.seqs, p.counts, b, p.tokens);
  if (i >= c) return;
  const int see = kv4_visible(n, c, i, p.causal), d = threadIdx.x;
  q[d] = static_cast<float>(
      static_cast<const T*>(p.q.ptr)[b * p.q.sb + i * p.q.st + hq * p.q.sh + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int base = 0; base < see; base += kKv4SimpleThreads) {
    const int slot = base + d;
    float x = -INFINITY;
    if (slot < see) {
      const long long page = kv4_page(p.pool, p.seqs, b, slot);
      if (page < 0) {
        kv4_report(p.seqs, kStatusKv4BadPage);
      } else {
        const uint8_t* half = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
        x = 0.f;
        for (int ch = 0; ch < kKv4Dim; ++ch)
          x += q[ch] * kv4_value_at(half, p.pool.ng, slot & 15, ch, false);
        x *= p.scale_log2;
      }
    }
    float top = x;
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if ((d & 31) == 0) red[d >> 5] = top;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float base_m = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - base_m);
    prob[d] = exp2f(x - base_m);
    __syncthreads();
    l *= a;
    o *= a;
    m = mn;
    for (int j = 0; j < min(kKv4SimpleThreads, see - base); ++j) {
      const float w = prob[j];
      const long long page = kv4_page(p.pool, p.seqs, b, base + j);
      if (page < 0) continue;
      l += w;
      const uint8_t* half = p.pool.pages + kv4_block_offset(p.pool, page, h, base + j) +
                            kv4_half_bytes(p.pool.ng);
      o += w * kv4_value_at(half, p.pool.ng, (base + j) & 15, d, true);
    }
    __syncthreads();
  }
  static_cast<T*>(p.o.ptr)[b * p.o.sb + i * p.o.st + hq * p.o.sh + d] =
      static_cast<T>(l == 0.f ? 0.f : o / l);
  if (d == 0) {
    const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
    if (p.lse != nullptr) p.lse[b * p.lse_sb + hq * p.lse_sh + i] = lse2 * 0.69314718055994531f;
    if (p.row_lse != nullptr)
      p.row_lse[(static_cast<long long>(b) * p.tokens + i) * p.heads_q + hq] = lse2;
  }
}

// One thread a (sequence, head, slot): the weight it received from every row.
template <typename T>
__global__ void __launch_bounds__(kKv4SimpleThreads) kv4_simple_weights_kernel(Kv4AttnParams p) {
  const int bh = blockIdx.y, h = bh % p.pool.heads, b = bh / p.pool.heads;
  const int n = kv4_length(p.pool, p.seqs, b), c = kv4_count(p.seqs, p.counts, b, p.tokens);
  const int group = p.heads_q / p.pool.heads;
  for (long long slot = blockIdx.x * kKv4SimpleThreads + threadIdx.x; slot < n;
       slot += static_cast<long long>(gridDim.x) * kKv4SimpleThreads) {
    const long long page = kv4_page(p.pool, p.seqs, b, slot);
    if (page < 0) continue;
    const uint8_t* half = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
    float sum = 0.f;
    for (int i = 0; i < c; ++i) {
      if (slot >= kv4_visible(n, c, i, p.causal)) continue;
      for (int g = 0; g < group; ++g) {
        const int hq = h * group + g;
        const T* q = static_cast<const T*>(p.q.ptr) + b * p.q.sb + i * p.q.st + hq * p.q.sh;
        float x = 0.f;
        for (int ch = 0; ch < kKv4Dim; ++ch)
          x += static_cast<float>(q[ch]) * kv4_value_at(half, p.pool.ng, slot & 15, ch, false);
        sum += exp2f(x * p.scale_log2 -
                     p.row_lse[(static_cast<long long>(b) * p.tokens + i) * p.heads_q + hq]);
      }
    }
    float* w = p.pool.weights + kv4_token_index(p.pool, page, h, slot);
    *w = p.decay == 0.f ? sum : p.decay * *w + sum;
  }
}

}  // namespace llmfa
