// Writing tokens into the 4-bit cache and reading them back.
//
// Over a group of channels, lo = min(0, x) and hi = max(0, x):
//   scale = bf16((hi - lo) / 15)     zero = clamp(round(-lo / scale), 0, 15)
//   code  = clamp(round(x / scale) + zero, 0, 15)       (halves to even)
// The range always takes in 0, so zero is an integer code and 0 is held
// exactly. A group with an infinity, a NaN or a range past fp32 is stored with
// a NaN scale: whoever reads it gets NaN, not a wrong number.
//
// The rounding is exact. x has at most 11 significant bits and scale 8, so
// x / scale is either a half-integer or at least 2^-12 away from one. The
// kernel takes x * (1 / scale), within 2^-19 of the quotient for |x / scale|
// <= 16, and adds 768 in one fused step, which rounds to a multiple of 2^-14:
// half-integers come back exactly, nothing else can reach one, and no divide
// is needed per value.
//
// Both kernels move bytes: 512 of a token's head on one side, 136 to 160 of
// codes and pairs on the other. A thread takes 8 channels (one 16-byte access)
// of the key and the value, 16 threads a token's head.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4_layout.cuh"

namespace llmfa {

constexpr int kKv4QuantThreads = 256;
constexpr int kKv4RowThreads = 16;  // threads of a token's head

struct Kv4RowView {  // [batch, tokens, heads, 128], element strides
  void* ptr;
  long long sb, st, sh;
};

template <typename T>
struct Kv4Type;
template <>
struct Kv4Type<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Kv4Type<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

// Scale, its reciprocal and zero of a group from its lo and hi.
struct Kv4Pair {
  float scale, inv, zero;
  uint32_t word;
};
__device__ __forceinline__ float kv4_snap(float x, float inv) {
  return __fadd_rn(__fmaf_rn(x, inv, 768.f), -768.f);
}
__device__ __forceinline__ Kv4Pair kv4_pair(float lo, float hi) {
  Kv4Pair p;
  float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
  // lo and hi skip NaN only in part (see kv4_range): any NaN or infinity shows in hi - lo
  if (!(s < __int_as_float(0x7f800000))) s = __int_as_float(0x7fc00000);
  // Below 2^-120 the reciprocal nears the end of fp32's range: such a group counts as zeros.
  if (s < 0x1p-120f) s = 0.f;
  p.scale = s;
  p.inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  p.zero = fminf(fmaxf(rintf(kv4_snap(-lo, p.inv)), 0.f), 15.f);
  p.word = (__float_as_uint(s) >> 16) | (__float_as_uint(p.zero) & 0xffff0000u);
  return p;
}
// 8 values -> 8 codes, low bits first.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], const Kv4Pair& p) {
  uint32_t w = 0;
  const int zero = static_cast<int>(p.zero);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // round to an integer by adding 1.5 * 2^23: halves to even, before zero is added
    const int r = __float_as_int(__fadd_rn(kv4_snap(x[i], p.inv), 12582912.f)) - 0x4B400000;
    const int u = min(max(r + zero, 0), 15);
    w |= static_cast<uint32_t>(u) << (4 * i);
  }
  return w;
}
// lo and hi of a group over the 16 / NG threads that hold it; NaN reaches both.
template <int NG>
__device__ __forceinline__ void kv4_range(const float (&x)[8], float& lo, float& hi) {
  lo = 0.f;
  hi = 0.f;
  float bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] * 0.f;  // NaN for NaN and infinities
  }
  hi += bad;
#pragma unroll
  for (int d = 1; d < kKv4RowThreads / NG; d <<= 1) {
    const float l = __shfl_xor_sync(0xffffffffu, lo, d), h = __shfl_xor_sync(0xffffffffu, hi, d);
    lo = fminf(lo, l);
    hi = h != h ? h : hi != hi ? hi : fmaxf(hi, h);
  }
}

struct Kv4AppendParams {
  Kv4Pool pool;
  Kv4Seqs seqs;
  Kv4RowView k, v;
  const int32_t* counts;  // new tokens of a sequence, or null
  const int32_t* seen;    // position of its first new token, or null: its length
  int tokens;
};

// One 16-thread row a (sequence, token, head); heads run fastest, as in memory.
template <typename T, int NG>
__global__ void __launch_bounds__(kKv4QuantThreads) kv4_append_kernel(Kv4AppendParams p) {
  const long long row = (static_cast<long long>(blockIdx.x) * kKv4QuantThreads + threadIdx.x) /
                        kKv4RowThreads;
  const int w = threadIdx.x % kKv4RowThreads;  // natural word: channels 8w .. 8w + 7
  const int heads = p.pool.heads;
  const long long rows = static_cast<long long>(p.seqs.batch) * p.tokens * heads;
  bool live = row < rows;
  const int h = live ? static_cast<int>(row % heads) : 0;
  const long long bt = live ? row / heads : 0;
  const int t = static_cast<int>(bt % p.tokens), b = static_cast<int>(bt / p.tokens);
  long long page = -1, slot = 0;
  if (live) {
    live = t < kv4_count(p.seqs, p.counts, b, p.tokens);
    slot = static_cast<long long>(p.seqs.lengths[b]) + t;
    if (live) {
      page = kv4_page(p.pool, p.seqs, b, slot);
      if (page < 0) kv4_report(p.seqs, kStatusKv4BadPage);
      live = page >= 0;
    }
  }
  uint4 raw[2] = {};
  if (live) {
    const long long at[2] = {b * p.k.sb + t * p.k.st + h * p.k.sh,
                             b * p.v.sb + t * p.v.st + h * p.v.sh};
    raw[0] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.k.ptr) + at[0] + 8 * w);
    raw[1] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.ptr) + at[1] + 8 * w);
  }
  uint32_t code[2], pair[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float x[8];
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&raw[side]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Kv4Type<T>::unpack(r[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    float lo, hi;
    kv4_range<NG>(x, lo, hi);
    const Kv4Pair q = kv4_pair(lo, hi);
    code[side] = kv4_codes(x, q);
    pair[side] = q.word;
  }
  // Values are stored by half-words: natural half-words 2w and 2w + 1 are k = w / 4, g = 2 (w % 4)
  // and g + 1. Threads w and w ^ 4 (k and k ^ 1) trade halves, so that each writes one word.
  const bool odd = (w & 4) != 0;
  const uint32_t give = odd ? code[1] & 0xffffu : code[1] >> 16;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 4);
  const uint32_t vword = odd ? (got | (code[1] & 0xffff0000u)) : ((code[1] & 0xffffu) | (got << 16));
  if (!live) return;
  uint8_t* block = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
  const int tok = static_cast<int>(slot & 15);
  uint8_t* vblock = block + kv4_half_bytes(NG);
  reinterpret_cast<uint32_t*>(block + tok * kKv4RowBytes)[kv4_key_word(w)] = code[0];
  // even k: g = 2 (w % 4), halves k, k + 1; odd k: g + 1, halves k - 1, k
  const int g = 2 * (w & 3) + (odd ? 1 : 0), k = (w >> 2) & ~1;
  reinterpret_cast<uint32_t*>(vblock + tok * kKv4RowBytes)[g * 2 + k / 2] = vword;
  constexpr int kGroupThreads = kKv4RowThreads / NG;
  if (w % kGroupThreads == 0) {
    const int at = tok * NG + w / kGroupThreads;
    reinterpret_cast<uint32_t*>(block + kKv4Block * kKv4RowBytes)[at] = pair[0];
    reinterpret_cast<uint32_t*>(vblock + kKv4Block * kKv4RowBytes)[at] = pair[1];
  }
  if (w == 0) {
    const long long i = kv4_token_index(p.pool, page, h, slot);
    p.pool.positions[i] = (p.seen != nullptr ? p.seen[b] : p.seqs.lengths[b]) + t;
    p.pool.weights[i] = 0.f;
  }
}

struct Kv4ExpandParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths: first slot of each sequence to read
  Kv4RowView k, v;
  const int32_t* counts;
  int tokens;
};

__device__ __forceinline__ float2 kv4_scale_zero(uint32_t pair) {
  return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint4 kv4_decode8(uint32_t codes, uint32_t pair) {
  const float2 sz = kv4_scale_zero(pair);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = Kv4Type<T>::pack(sz.x * (static_cast<float>((codes >> (8 * i)) & 15u) - sz.y),
                            sz.x * (static_cast<float>((codes >> (8 * i + 4)) & 15u) - sz.y));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// The inverse of kv4_append_kernel; rows past a sequence's count are zeros.
template <typename T, int NG>
__global__ void __launch_bounds__(kKv4QuantThreads) kv4_expand_kernel(Kv4ExpandParams p) {
  const long long row = (static_cast<long long>(blockIdx.x) * kKv4QuantThreads + threadIdx.x) /
                        kKv4RowThreads;
  const int w = threadIdx.x % kKv4RowThreads;
  const int heads = p.pool.heads;
  if (row >= static_cast<long long>(p.seqs.batch) * p.tokens * heads) return;
  const int h = static_cast<int>(row % heads);
  const long long bt = row / heads;
  const int t = static_cast<int>(bt % p.tokens), b = static_cast<int>(bt / p.tokens);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (t < kv4_count(p.seqs, p.counts, b, p.tokens)) {
    const long long slot = static_cast<long long>(p.seqs.lengths[b]) + t;
    const long long page = kv4_page(p.pool, p.seqs, b, slot);
    if (page < 0) {
      kv4_report(p.seqs, kStatusKv4BadPage);
    } else {
      const uint8_t* block = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
      const uint8_t* vblock = block + kv4_half_bytes(NG);
      const int tok = static_cast<int>(slot & 15), at = tok * NG + w / (kKv4RowThreads / NG);
      const uint32_t kc =
          reinterpret_cast<const uint32_t*>(block + tok * kKv4RowBytes)[kv4_key_word(w)];
      const uint16_t* vr = reinterpret_cast<const uint16_t*>(vblock + tok * kKv4RowBytes);
      const uint32_t vc = vr[kv4_value_half(2 * w)] |
                          (static_cast<uint32_t>(vr[kv4_value_half(2 * w + 1)]) << 16);
      k = kv4_decode8<T>(kc, reinterpret_cast<const uint32_t*>(block + kKv4Block * kKv4RowBytes)[at]);
      v = kv4_decode8<T>(vc, reinterpret_cast<const uint32_t*>(vblock + kKv4Block * kKv4RowBytes)[at]);
    }
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(p.k.ptr) + b * p.k.sb + t * p.k.st + h * p.k.sh + 8 * w) = k;
  *reinterpret_cast<uint4*>(static_cast<T*>(p.v.ptr) + b * p.v.sb + t * p.v.st + h * p.v.sh + 8 * w) = v;
}

}  // namespace llmfa
