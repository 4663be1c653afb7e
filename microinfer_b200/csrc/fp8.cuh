// The 8-bit paged KV cache: its page layout and the conversions in and out.
//
// K and V are held in 8-bit floating point (e4m3: sign, 4 bits of exponent, 3 of mantissa; largest 448, smallest
// 2^-9, 0x7f and 0xff not a number) with one power-of-two scale for every block of 16 tokens and kv head.  A
// pool is uint8 [num_blocks][num_kv_heads][block_size / 16][16 * D + 16]; the last dimension is a group of 16 tokens
// of one kv head, its codes in parts of 64 dims (w = 64; a last part of 32 where D is an odd multiple of 32):
//   K   [16 tokens][w]
//   V   [2 halves][8][4 pairs][w / 8 dims][2 tokens]   token = 8 half + 2 pair + last, dim = w / 8 * second + fourth
// then 16 bytes: the scale byte b, 2^(b - 127), 0 for zero, and 15 that are zero.
// A group is contiguous, a multiple of 16 bytes.  A part of K or V is what the 32 lanes of a warp want as MMA
// operands, in the order of the lanes: 16 bytes of lane (g, t) are 16 dims of K's token g, or 8 dims of the pair t of V's
// tokens, whose two bytes side by side become one f16 pair, the two k-slots of a register.
//
// Powers of two: a division by the scale is exact, so codes depend on the group's scale alone, and where a later
// token raises it the codes that are there lose nothing but what becomes subnormal (below 2^-14 of the group's largest).
// One exponent for a whole group is also what keeps the scale out of the products: it is a factor of 16 keys' scores
// and of 16 keys' p, not of the elements.
#pragma once

#include "common.cuh"

namespace mi {

constexpr int kF8Group = 16;  // tokens that share a scale
constexpr int kF8Tail = 16;   // bytes after a group's codes, the scale first
constexpr uint32_t kF8Largest = 246;  // scale byte: 448 * 2^119 is below fp32's and bf16's largest

__host__ __device__ constexpr int f8_group_bytes(int head_dim) { return kF8Group * head_dim + kF8Tail; }

// Place of 8 dims from 8 * octet on in a group: K's of token 0 (tokens are `row` bytes apart), V's of pair 0 of half 0
// (pairs `pair` bytes apart, halves `half`); in a last part of 32 dims V's dims 4 to 7 are `split` bytes behind the first four.
struct F8Place {
  int k, row, v, pair, half, split;
};
__device__ __forceinline__ F8Place f8_place(int octet, int head_dim) {
  const int part = octet >> 3, base = part * 64 * kF8Group, i = octet & 7;
  F8Place r;
  if ((part + 1) * 64 <= head_dim) {
    r.k = base + i * 8, r.row = 64;
    r.v = base + i * 64, r.pair = 16, r.half = 512, r.split = 8;
  } else {
    r.k = base + i * 8, r.row = 32;
    r.v = base + i * 64, r.pair = 8, r.half = 256, r.split = 32;
  }
  return r;
}

// Four codes of a word as f16 pairs (exact): bytes 0 and 1, bytes 2 and 3.
__device__ __forceinline__ void f8_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("{ .reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h; }"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// Four codes of a word, unscaled, as floats.
__device__ __forceinline__ void f8_to_f32(uint32_t w, float (&x)[4]) {
  uint32_t r[2];
  f8_to_f16(w, r[0], r[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// Four floats to codes (a in the lowest byte): to nearest, ties to even, saturating at 448; NaN stays.
__device__ __forceinline__ uint32_t f8_encode4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{ .reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h}; }"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Whether one of a word's codes is a NaN.
__device__ __forceinline__ bool f8_any_nan(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// The softmax's scale (log2 domain) taken apart: its magnitude is mantissa * 2^exponent, the mantissa in [1, 2) or an infinity,
// and q is multiplied by its sign, so that the largest product is the largest score.  Of a scale of 0 or NaN the
// sign is 0 or NaN, which makes every score that, and the rest stands for 1.
struct F8Scale {
  float mantissa, sign;
  int exponent;
};
__host__ __device__ __forceinline__ F8Scale f8_softmax_scale(float scale) {
  F8Scale r = {1.f, scale, 0};
  const float a = fabsf(scale);
  if (a > 0.f) {
    r.sign = scale < 0.f ? -1.f : 1.f;
    r.mantissa = a;
    if (a < INFINITY) {
      r.mantissa = 2.f * frexpf(a, &r.exponent);
      --r.exponent;
    }
  }
  return r;
}

// 2^(b - 127), 0 for 0.
__device__ __forceinline__ float f8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte that a largest magnitude (as bits of a finite float) needs.
__device__ __forceinline__ uint32_t f8_byte_for(uint32_t top) {
  const int b = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8
  return top == 0 ? 0u : static_cast<uint32_t>(min(max(b, 1), static_cast<int>(kF8Largest)));
}

}  // namespace mi
