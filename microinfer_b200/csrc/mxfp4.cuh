// The 4-bit paged KV cache: its page layout and the conversions in and out.
//
// K and V are held in microscaled 4-bit floating point (MXFP4): e2m1 codes
// (sign, then 0, 0.5, 1, 1.5, 2, 3, 4 or 6) with one power-of-two scale for
// every 32 of them along the head dimension, 4.25 bits per element.  A pool is
// uint8 [num_blocks][num_kv_heads][block_size / 16][D / 32 * 272]; the last
// dimension is a group of 16 tokens of one kv head:
//   codes   [D / 32][16 tokens][16 bytes]   element 2j in the low nibble of byte j
//   scales  [16 tokens][D / 32]             byte e: 2^(e - 127); 0: zero; 255: NaN
// A group is contiguous (1088 bytes at D = 128), so one bulk copy brings it,
// and 8 tokens of one 32-element block are 128 consecutive bytes, so the
// 8 x 16-byte rows of an ldmatrix touch every shared-memory bank once.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace mi {

constexpr int kMxBlock = 32;   // elements that share a scale
constexpr int kMxGroup = 16;   // tokens of a group
constexpr int kMxBlockBytes = kMxGroup * 16;                // codes of one block of a group
constexpr int kMxBytes = kMxBlockBytes + kMxGroup;          // codes and scales of one block

__host__ __device__ constexpr int mx_group_bytes(int head_dim) {
  return head_dim / kMxBlock * kMxBytes;
}

// n / d by a multiplication, n below 2^31.
struct FastDiv {
  uint32_t mul;
  int shift;
  explicit FastDiv(uint32_t d) {
    shift = 31;
    while ((uint64_t{1} << (shift - 31)) < d) ++shift;
    mul = static_cast<uint32_t>(((uint64_t{1} << shift) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>(static_cast<uint64_t>(n) * mul >> shift);
  }
};

__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

// Blocks that 16-bit rows of type T cannot stand for in a product with zeros: NaN blocks of V (0 * NaN reaches rows that do
// not see the key; one of K only meets its own scores), and those of K and V past fp16, which ends at
// 65504 = 3.998 * 2^14.
template <typename T>
constexpr uint32_t mx_apart_from = std::is_same<T, __half>::value ? 127 + 14 : 255;
template <typename T>
__device__ __forceinline__ bool mx_apart(bool value, uint32_t byte) {
  return byte >= mx_apart_from<T> && (value || (std::is_same<T, __half>::value && byte != 255u));
}

// Eight codes of a word, in element order, as four f16 pairs (exact).
// All four bytes of the unpacked word are converted here: where the statement converts only one of them, nvcc
// 12.9 gives 0 for every byte.  In this form all 256 bytes are right in every place, whichever results are used and
// whether the word is loaded, masked or a byte extended by zeros.
__device__ __forceinline__ void mx_codes_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{ .reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3; }"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}

// Eight codes of a word times `scale`, as floats.
__device__ __forceinline__ void mx_codes_to_f32(uint32_t w, float scale, float (&x)[8]) {
  uint32_t r[4];
  mx_codes_to_f16(w, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
    x[2 * i] = f.x * scale;
    x[2 * i + 1] = f.y * scale;
  }
}

// Four floats -> 16 bits of codes (a in the lowest nibble), twice: round to
// nearest, ties to even, saturating at 6.
__device__ __forceinline__ uint32_t mx_encode4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{ .reg .b8 b0, b1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "mov.b32 %0, {b0, b1, b0, b1}; }"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

}  // namespace mi
