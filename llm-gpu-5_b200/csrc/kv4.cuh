// The 4-bit key/value cache: layout, and the arithmetic of one group, shared by the store, load,
// decode and eviction kernels.
//
// A cached row holds the D values of one (sequence, head, position) in groups of g = min(D, 64).  A
// group keeps s = f16((max - min) / 15) and m = f16(min), both computed in float32 (the division as a
// product with the float32 nearest to 1/15), and per value the code n in 0..15 nearest to (x - m) / s in exact arithmetic (ties to even); it stands for n*s + m.
//   codes  [2][B][NH][cap][D / 2] bytes   (0 keys, 1 values; element d = 2i in the low nibble of byte i)
//   params [2][B][NH][cap][D / g] half2   (s, m)
// Rows of one (sequence, head) are contiguous, so that a run of keys is one contiguous copy; the other
// axes are strided, in rows, with the same strides for codes and params.  cap and the strides are
// multiples of 16 rows, which keeps every 16th row 16-byte aligned in both arrays for every D.
#pragma once

#include "common.cuh"
#include <cuda_fp16.h>

namespace attn {

constexpr int KV4_ALIGN_ROWS = 16;

__host__ __device__ constexpr int kv4_group(int D) { return D < 64 ? D : 64; }
__host__ __device__ constexpr int kv4_groups(int D) { return D / kv4_group(D); }
inline bool kv4_head_dim_ok(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }

struct Kv4View {
  uint8_t* codes;
  __half2* params;
  int64_t si, sb, sh;  // strides in rows: keys -> values, sequence, head
  int cap;             // rows per (sequence, head)
};

// Rows of `len` units (elements, or cached rows) along up to three strided axes.  They are apart where every stride
// is at least the span of the axes inside it, so that CTAs may write them side by side; a layout whose rows miss one
// another in some other way counts as overlapping.
struct RowSet {
  int64_t n[3] = {1, 1, 1}, s[3] = {0, 0, 0};  // axes of more than one entry, the largest stride first
  int64_t len, span;                           // span: from the first row to the end of the last
  bool apart = true;
  RowSet(int64_t len_, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2 = 1, int64_t s2 = 0) : len(len_), span(len_) {
    const int64_t ns[3] = {n0, n1, n2}, ss[3] = {s0, s1, s2};
    int axes = 0;
    for (int i = 0; i < 3; ++i) {
      if (ns[i] <= 1) continue;
      int at = axes++;
      for (; at > 0 && s[at - 1] < ss[i]; --at) { n[at] = n[at - 1]; s[at] = s[at - 1]; }
      n[at] = ns[i];
      s[at] = ss[i];
    }
    for (int i = axes - 1; i >= 0 && apart; --i) {
      apart = s[i] >= span && s[i] <= ((int64_t)1 << 52) / n[i] - span;  // (2^52 units are more than any memory)
      if (apart) span += (n[i] - 1) * s[i];
    }
  }
  // Whether rows of `bytes` bytes a unit at p share memory with those of b at q (both apart).
  bool meets(const void* p, const RowSet& b, const void* q, int64_t bytes) const {
    const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(p) - reinterpret_cast<intptr_t>(q));
    if (d >= b.span * bytes || -d >= span * bytes) return false;
    for (int64_t i = 0; i < n[0]; ++i)
      for (int64_t j = 0; j < n[1]; ++j)
        for (int64_t k = 0; k < n[2]; ++k) {
          const int64_t first = d + (i * s[0] + j * s[1] + k * s[2]) * bytes;  // of this row, from q on
          int64_t left = first + len * bytes - 1, at = 0;                       // the last row of b that starts by then
          if (left < 0) continue;
          for (int x = 0; x < 3; ++x) {
            if (b.n[x] <= 1) continue;
            const int64_t stride = b.s[x] * bytes, c = left / stride < b.n[x] - 1 ? left / stride : b.n[x] - 1;
            at += c * stride;
            left -= c * stride;
          }
          if (at + b.len * bytes > first) return true;
        }
    return false;
  }
};

// Checks shared by the entry points that take a cache.
int kv4_check(const char* fn, const Kv4View& c, int B, int NH, int D);

// An int32 per sequence: base[b] + add, or add alone when base is NULL.
__device__ __forceinline__ int64_t seq_value(const int* base, int b, int add) {
  return (base ? (int64_t)base[b] : 0) + add;
}

// Rows of sequence b: lengths[b] clamped to 0..most, or most when lengths is NULL.
__device__ __forceinline__ int seq_length(const int* lengths, int b, int most) {
  return lengths ? min(max(lengths[b], 0), most) : most;
}

// n / d for 0 <= n < 2^31 as a multiplication by m = ceil(2^(31 + k) / d), k = ceil(log2 d): n m / 2^(31 + k)
// exceeds n / d by less than n / 2^31 / d < 1 / d.
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ void set(uint32_t divisor) {
    d = divisor;
    shift = 0;
    while ((1u << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> (31 + shift)); }
};

// The code of x in a group (s, m): the n in 0..15 nearest to (x - m) / s, ties to even, decided in
// exact arithmetic.  x - m is split into its float32 rounding d and the rounding's error e (Knuth's
// two-sum), and the borders (n +- 1/2) s are exact in float32 (5 + 11 bits); a division can only
// place a value near a border on the wrong side of it, which the comparisons put right.
__device__ __forceinline__ uint32_t kv4_code_exact(float x, float s, float m, float inv) {
  const float d = __fsub_rn(x, m);
  const float bb = __fsub_rn(d, x);
  const float e = __fadd_rn(__fsub_rn(x, __fsub_rn(d, bb)), -__fadd_rn(m, bb));
  float n = fminf(fmaxf(rintf(__fmul_rn(d, inv)), 0.f), 15.f);
  const float hi = __fmul_rn(n + 0.5f, s), lo = __fmul_rn(n - 0.5f, s);
  const bool odd = ((int)n & 1) != 0;
  if (d > hi || (d == hi && (e > 0.f || (e == 0.f && odd)))) n += 1.f;
  else if (d < lo || (d == lo && (e < 0.f || (e == 0.f && odd)))) n -= 1.f;
  return (uint32_t)fminf(fmaxf(n, 0.f), 15.f);
}

// The codes of eight values as one word, inv = 1 / s to 2^-22.  t = 15 sat((x - m) inv / 15) + 0 in float32 is
// within 15 * 5 * 2^-24 < 5e-6 of the exact quotient clamped to 0..15 (which decides alike), so its nearest
// integer is the code unless t lies within 1e-5 of a border; such a value is decided again exactly
// (bfloat16 values are so coarse that one in 1,250 lies on a border, and a third of the warps hold one).
// The saturation, the rounding (adding 1.5 * 2^23 leaves the integer in the low bits) and the packing
// (w * 16 + bits, the constant part taken off at the end) all run on the multiply-add pipe.
__device__ __forceinline__ uint32_t kv4_word(const float (&x)[8], float s, float m, float inv) {
  constexpr float MAGIC = 12582912.f;
  constexpr uint32_t MAGIC_BITS = 0x4b400000u;
  const float inv15 = __fmul_rn(inv, 1.f / 15.f);
  uint32_t w = 0;
  float far = 0.f;
  auto place = [&](float v, float& r) {  // distance from the nearest integer, which is left in r's low bits
    const float t = __saturatef(__fmul_rn(__fsub_rn(v, m), inv15));
    r = __fmaf_rn(t, 15.f, MAGIC);
    return fabsf(__fmaf_rn(t, 15.f, -__fsub_rn(r, MAGIC)));
  };
#pragma unroll
  for (int i = 7; i >= 0; i -= 2) {
    float r0, r1;
    const float f0 = place(x[i], r0), f1 = place(x[i - 1], r1);
    asm("max.f32 %0, %0, %1, %2;" : "+f"(far) : "f"(f0), "f"(f1));
    w = (w * 16u + __float_as_uint(r0)) * 16u + __float_as_uint(r1);
  }
  w -= (uint32_t)(MAGIC_BITS * 0x11111111ull);
  if (far > 0.49999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float r;
      if (place(x[i], r) > 0.49999f) w = (w & ~(15u << (4 * i))) | kv4_code_exact(x[i], s, m, inv) << (4 * i);
    }
  }
  return s > 0.f ? w : 0u;
}

// The numbers n s + m of a word's eight codes, each rounded once (n s is exact: 4 + 11 bits).  A code
// is made a float32 where it stands: its bits in the mantissa of 2^23, which is then taken off; that leaves
// n * 16^k, and s * 16^-k is exact.
__device__ __forceinline__ void kv4_values(uint32_t w, float s, float m, float (&x)[8]) {
  constexpr float BIG = 8388608.f;
  float sk = s;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t mask = 15u << (4 * k);
    x[k] = __fmaf_rn(__uint_as_float((w & mask) | 0x4b000000u) - BIG, sk, m);
    x[k + 4] = __fmaf_rn(__uint_as_float(((w >> 16) & mask) | 0x4b000000u) - BIG, sk, m);
    sk *= 0.0625f;
  }
}

}  // namespace attn
