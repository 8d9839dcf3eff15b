// Writing tokens into the 4-bit cache and reading them back.
//
// Over a group of channels, lo = min(0, x) and hi = max(0, x):
//   scale = bf16((hi - lo) / 15)     zero = clamp(round(-lo / scale), 0, 15)
//   code  = clamp(round(x / scale) + zero, 0, 15)       (halves to even)
// The range always takes in 0, so zero is an integer code and 0 is held
// exactly. A group with an infinity or a NaN is stored with a NaN scale: whoever
// reads it gets NaN, not a wrong number.
//
// The rounding is exact. x has at most 11 significant bits and scale 8, so
// x / scale is either a half-integer or at least 2^-12 away from one. The
// kernel takes x * (1 / scale), within 2^-19 of the quotient for |x / scale|
// <= 16, and adds 768 in one fused step, which rounds to a multiple of 2^-14:
// half-integers come back exactly, nothing else can reach one, and no divide
// is needed per value. Adding 1.5 * 2^23 - 768 then rounds to an integer,
// halves to even, in the low bits. As rounding is monotone and odd, no code
// falls below 0; only the upper end has to be clamped.
//
// Both kernels move bytes: 512 of a token's head on one side, 136 to 160 of
// codes and pairs on the other. What would bound them otherwise is
// instructions: a thread takes 16 channels of the key and the value, so that
// the addresses of a token's head are worked out by 8 threads; ranges are taken
// on packed pairs; codes become numbers as fp16 integers. Measured: 8192 tokens
// of 32 heads, groups of 32, in and back out: 38 + 31 us, 4.7 and 5.7 TB/s of
// 6.6; with 8 channels a thread and 64-bit divisions in front it was 83 + 49.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "kv4_layout.cuh"

namespace llmfa {

constexpr int kKv4QuantThreads = 256;
constexpr int kKv4RowThreads = 8;  // threads of a token's head, 16 channels each

struct Kv4RowView {  // [batch, tokens, heads, 128], element strides
  void* ptr;
  long long sb, st, sh;
};

// Division of numbers below 2^31 by a d fixed before the launch.
struct Kv4Div {
  uint32_t mul, shift, d;
  Kv4Div() = default;
  __host__ __device__ explicit Kv4Div(uint32_t by) : mul(0), shift(0), d(by) {
    while ((uint64_t(1) << shift) < by) ++shift;
    mul = static_cast<uint32_t>((((uint64_t(1) << shift) - by) << 32) / by + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return (__umulhi(n, mul) + n) >> shift;
  }
#endif
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
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {  // NaN if either is
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
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
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};

__device__ __forceinline__ float2 kv4_scale_zero(uint32_t pair) {
  return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}

// Scale, its reciprocal and zero of a group from its lo and hi.
struct Kv4Pair {
  float inv;
  int zero;
  uint32_t word;
};
// x / 15, correctly rounded: the product with 1/15 and one correction by its exact remainder
// (Markstein's scheme; a test compares it with the quotient for every mantissa, as host code).
__host__ __device__ __forceinline__ float kv4_fifteenth(float x) {
  constexpr float c = 1.f / 15.f;
#ifdef __CUDA_ARCH__
  const float q = __fmul_rn(x, c);
  return __fmaf_rn(__fmaf_rn(-15.f, q, x), c, q);
#else
  const float q = x * c;
  return std::fma(std::fma(-15.f, q, x), c, q);
#endif
}
__device__ __forceinline__ Kv4Pair kv4_pair(float lo, float hi) {
  Kv4Pair p;
  // of halves: hi - lo itself may pass fp32's range
  const float span = __fmaf_rn(hi, 0.5f, -0.5f * lo);
  float s = 2.f * __bfloat162float(__float2bfloat16_rn(kv4_fifteenth(span)));
  // a NaN or an infinity in the group shows in their difference
  if (!(span < __int_as_float(0x7f800000))) s = __int_as_float(0x7fc00000);
  // Below 2^-120 the reciprocal nears the end of fp32's range: such a group counts as zeros.
  if (s < 0x1p-120f) s = 0.f;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  p.inv = s > 0.f ? inv : 0.f;
  const float r = __fadd_rn(__fmaf_rn(-lo, p.inv, 768.f), 12582912.f - 768.f);
  const float zero = fminf(fmaxf(__fadd_rn(r, -12582912.f), 0.f), 15.f);
  p.zero = __float_as_int(__fadd_rn(zero, 12582912.f)) - 0x4B400000;
  p.word = __byte_perm(__float_as_uint(s), __float_as_uint(zero), 0x7632);
  return p;
}
// 8 values -> 8 codes, low bits first.
template <typename T>
__device__ __forceinline__ uint32_t kv4_codes(const uint4& raw, const Kv4Pair& p) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
  const int base = p.zero - 0x4B400000;
  uint32_t w = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const float2 x = Kv4Type<T>::unpack(r[i]);
#pragma unroll
    for (int k = 1; k >= 0; --k) {
      const float v = __fadd_rn(__fmaf_rn(k ? x.y : x.x, p.inv, 768.f), 12582912.f - 768.f);
      w = w * 16 + min(__float_as_int(v) + base, 15);
    }
  }
  return w;
}
// lo = min(0, x) and hi = max(0, x) of a group, over the 8 / NG threads that hold it; a NaN in it
// makes both NaN. From thread to thread they go as one word, (lo, -hi): both are minima then.
template <typename T, int NG>
__device__ __forceinline__ float2 kv4_range(const uint4 (&raw)[2]) {
  using V = Kv4Type<T>;
  const uint32_t lo2 = V::min2(V::min2(V::min2(raw[0].x, raw[0].y), V::min2(raw[0].z, raw[0].w)),
                               V::min2(V::min2(raw[1].x, raw[1].y), V::min2(raw[1].z, raw[1].w)));
  const uint32_t hi2 = V::max2(V::max2(V::max2(raw[0].x, raw[0].y), V::max2(raw[0].z, raw[0].w)),
                               V::max2(V::max2(raw[1].x, raw[1].y), V::max2(raw[1].z, raw[1].w)));
  const uint32_t minus = hi2 ^ 0x80008000u;
  uint32_t both = V::min2(__byte_perm(lo2, minus, 0x5410), __byte_perm(lo2, minus, 0x7632));
  both = V::min2(both, 0u);
#pragma unroll
  for (int d = 1; d < kKv4RowThreads / NG; d <<= 1)
    both = V::min2(both, __shfl_xor_sync(0xffffffffu, both, d));
  const float2 f = V::unpack(both);
  return make_float2(f.x, -f.y);
}

struct Kv4AppendParams {
  Kv4Pool pool;
  Kv4Seqs seqs;
  Kv4RowView k, v;
  const int32_t* counts;  // new tokens of a sequence, or null
  const int32_t* seen;    // position of its first new token, or null: its length
  int tokens;
  Kv4Div heads;
};

// A thread's row: 8 threads a (token, head) of sequence blockIdx.y; heads run fastest, as in
// memory.
struct Kv4QuantRow {
  int b, t, h;
  bool live;
};
__device__ __forceinline__ Kv4QuantRow kv4_quant_row(const Kv4Div& heads, int tokens) {
  const uint32_t row = (blockIdx.x * kKv4QuantThreads + threadIdx.x) / kKv4RowThreads;
  const uint32_t t = heads.quotient(row);
  return {static_cast<int>(blockIdx.y), static_cast<int>(t), static_cast<int>(row - t * heads.d),
          t < static_cast<uint32_t>(tokens)};
}

template <typename T, int NG>
__global__ void __launch_bounds__(kKv4QuantThreads)
    kv4_append_kernel(const __grid_constant__ Kv4AppendParams p) {
  const Kv4QuantRow row = kv4_quant_row(p.heads, p.tokens);
  const int a = threadIdx.x % kKv4RowThreads;  // channels 16a .. 16a + 15: natural words 2a, 2a + 1
  const int b = row.b, t = row.t, h = row.h;
  const int held = p.seqs.lengths[b];
  const long long slot = static_cast<long long>(held) + t;
  bool live = row.live && t < kv4_count(p.seqs, p.counts, b, p.tokens);
  if (held < 0) {  // no slot to write behind
    kv4_report(p.seqs, kStatusKv4BadLength);
    live = false;
  }
  long long page = -1;
  uint4 raw[2][2] = {};
  if (live) {
    page = kv4_page(p.pool, p.seqs, b, slot);
    const uint4* k = reinterpret_cast<const uint4*>(static_cast<const T*>(p.k.ptr) + b * p.k.sb +
                                                    t * p.k.st + h * p.k.sh + 16 * a);
    const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.ptr) + b * p.v.sb +
                                                    t * p.v.st + h * p.v.sh + 16 * a);
    raw[0][0] = k[0];
    raw[0][1] = k[1];
    raw[1][0] = v[0];
    raw[1][1] = v[1];
    if (page < 0) kv4_report(p.seqs, kStatusKv4BadPage);
    live = page >= 0;
  }
  uint32_t code[2][2], pair[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const float2 range = kv4_range<T, NG>(raw[side]);
    const Kv4Pair q = kv4_pair(range.x, range.y);
    code[side][0] = kv4_codes<T>(raw[side][0], q);
    code[side][1] = kv4_codes<T>(raw[side][1], q);
    pair[side] = q.word;
  }
  // Values are stored by half-words: this thread's are k = a / 2 and g = 4 (a % 2) .. + 3 of the
  // natural k * 8 + g. Threads a and a ^ 2 (k and k ^ 1) trade halves, so that each writes two
  // whole words, of the g of its own word (a & 2) / 2.
  const bool odd = (a & 2) != 0;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, code[1][odd ? 0 : 1], 2);
  const uint32_t mine = code[1][odd ? 1 : 0];
  const uint32_t even_k = odd ? got : mine, odd_k = odd ? mine : got;
  if (!live) return;
  uint8_t* block = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
  const int tok = static_cast<int>(slot & 15);
  uint8_t* vblock = block + kv4_half_bytes(NG);
  uint32_t* krow = reinterpret_cast<uint32_t*>(block + tok * kKv4RowBytes);
  krow[kv4_key_word(2 * a)] = code[0][0];
  krow[kv4_key_word(2 * a + 1)] = code[0][1];
  uint32_t* vrow = reinterpret_cast<uint32_t*>(vblock + tok * kKv4RowBytes);
  const int g = 4 * (a & 1) + (odd ? 2 : 0), word = g * 2 + (a >> 2);
  vrow[word] = __byte_perm(even_k, odd_k, 0x5410);
  vrow[word + 2] = __byte_perm(even_k, odd_k, 0x7632);
  constexpr int kGroupThreads = kKv4RowThreads / NG;
  if (a % kGroupThreads == 0) {
    const int at = tok * NG + a / kGroupThreads;
    reinterpret_cast<uint32_t*>(block + kKv4Block * kKv4RowBytes)[at] = pair[0];
    reinterpret_cast<uint32_t*>(vblock + kKv4Block * kKv4RowBytes)[at] = pair[1];
  }
  if (a == 0) {
    const long long i = kv4_token_index(p.pool, page, h, slot);
    p.pool.positions[i] = (p.seen != nullptr ? p.seen[b] : held) + t;
    p.pool.weights[i] = 0.f;
  }
}

struct Kv4ExpandParams {
  Kv4Pool pool;
  Kv4Seqs seqs;  // lengths: first slot of each sequence to read
  Kv4RowView k, v;
  const int32_t* counts;
  int tokens;
  Kv4Div heads;
};

// 8 codes as fp16 integers less their zero (0x6400 + u is 1024 + u, and 1024 + 16 u in the next
// nibble), then fp32 times the scale: exact up to the one rounding to T.
template <typename T>
__device__ __forceinline__ uint4 kv4_decode8(uint32_t codes, uint32_t pair) {
  const float2 sz = kv4_scale_zero(pair);
  const __half2 zero = __float2half2_rn(1024.f + sz.y);
  const __half2 zero16 = __float2half2_rn(-64.f - sz.y);
  const __half2 sixteenth = __float2half2_rn(0.0625f);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // nibbles i and i + 4
    const uint32_t c = i < 2 ? codes : codes >> 8;
    uint32_t bits;
    if (i % 2 == 0) asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(bits) : "r"(c));
    else asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(bits) : "r"(c));
    const __half2 u = *reinterpret_cast<__half2*>(&bits);
    const float2 f = __half22float2(i % 2 == 0 ? __hsub2(u, zero) : __hfma2(u, sixteenth, zero16));
    x[i] = f.x * sz.x;
    x[i + 4] = f.y * sz.x;
  }
  return make_uint4(Kv4Type<T>::pack(x[0], x[1]), Kv4Type<T>::pack(x[2], x[3]),
                    Kv4Type<T>::pack(x[4], x[5]), Kv4Type<T>::pack(x[6], x[7]));
}

// The inverse of kv4_append_kernel; rows past a sequence's count are zeros.
template <typename T, int NG>
__global__ void __launch_bounds__(kKv4QuantThreads)
    kv4_expand_kernel(const __grid_constant__ Kv4ExpandParams p) {
  const Kv4QuantRow row = kv4_quant_row(p.heads, p.tokens);
  if (!row.live) return;
  const int a = threadIdx.x % kKv4RowThreads, b = row.b, t = row.t, h = row.h;
  uint4 k[2] = {}, v[2] = {};
  if (t < kv4_count(p.seqs, p.counts, b, p.tokens)) {
    const long long slot = static_cast<long long>(p.seqs.lengths[b]) + t;
    const long long page = kv4_page(p.pool, p.seqs, b, slot);
    if (page < 0) {
      kv4_report(p.seqs, kStatusKv4BadPage);
    } else {
      const uint8_t* block = p.pool.pages + kv4_block_offset(p.pool, page, h, slot);
      const uint8_t* vblock = block + kv4_half_bytes(NG);
      const int tok = static_cast<int>(slot & 15);
      const uint32_t* kr = reinterpret_cast<const uint32_t*>(block + tok * kKv4RowBytes);
      const uint16_t* vr = reinterpret_cast<const uint16_t*>(vblock + tok * kKv4RowBytes);
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(block + kKv4Block * kKv4RowBytes) + tok * NG;
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(vblock + kKv4Block * kKv4RowBytes) + tok * NG;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int w = a + 8 * i;
        const uint32_t vc = vr[kv4_value_half(2 * w)] |
                            (static_cast<uint32_t>(vr[kv4_value_half(2 * w + 1)]) << 16);
        k[i] = kv4_decode8<T>(kr[kv4_key_word(w)], kp[w * NG / 16]);
        v[i] = kv4_decode8<T>(vc, vp[w * NG / 16]);
      }
    }
  }
  // words a and a + 8: the 8 threads write 128 contiguous bytes at a time
  uint4* ko = reinterpret_cast<uint4*>(static_cast<T*>(p.k.ptr) + b * p.k.sb + t * p.k.st + h * p.k.sh + 8 * a);
  uint4* vo = reinterpret_cast<uint4*>(static_cast<T*>(p.v.ptr) + b * p.v.sb + t * p.v.st + h * p.v.sh + 8 * a);
  ko[0] = k[0];
  ko[8] = k[1];
  vo[0] = v[0];
  vo[8] = v[1];
}

}  // namespace llmfa
