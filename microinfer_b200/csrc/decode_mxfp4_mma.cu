// Paged decode over the 4-bit cache (layout: mxfp4.cuh) on the warp-level tensor cores: one query
// token per sequence, out = softmax(scale * K q) V, any type, head_dim and GQA group.
//
// Decode moves 4.25 bits per cached element and does 2 flops per element and
// query head on it, so the bound is HBM as long as turning codes into MMA
// operands stays cheap.  What makes it so:
//   - an e2m1 byte becomes an f16 pair in one instruction (cvt.rn.f16x2.e2m1x2);
//   - codes go into the MMA without their scales.  S^T = K Q^T is accumulated per
//     32-element block (two m16n8k16 steps) and the block's scale multiplies
//     the 16 keys x 8 queries in fp32: D / 32 multiplications per score instead of D;
//   - the scale of V depends on the key and the block, so it goes into P: for each block,
//     P_b[key, query] = p * 2^(scale - R_b) in f16, R_b a running reference of the block kept
//     with the accumulators.  p is held up by 2^12 (and m no more than 3 binades behind
//     the largest score), so P_b uses f16 from 2^15 down: a key 2^-19 of the largest keeps all its
//     bits even 7 binades below R_b, and nothing above 2^-30 is lost, which a long context with
//     one dominant key needs.  A group with a scale more than 7 binades below R_b, or above it
//     (or zero, or NaN) takes a slower path that raises R_b or runs the products in windows of
//     8 binades, so no spread of scales loses more.  R_b never falls within a segment: one token of V that is 2^6
//     above all later ones keeps them on that path (32 x 8192: 60 us, then 92; a zero block in
//     every group 119; scales over 23 binades 175);
//   - q is multiplied by a power of two that puts its largest element into
//     [2^14, 2^15) and converted to f16 (exact for bf16 down to 2^-28 of that element).
// No code is moved between lanes or interleaved.  An ldmatrix of 8 keys x 16 bytes gives each lane 8
// consecutive codes of its key: K's A fragments, with dims in an order that q follows.  The
// transposed one gives a lane two bytes of each of two keys, and each byte, two neighbouring dims of
// one key, is an A register of V^T whose two k-slots are (key, even dim) and (key, odd dim);
// the B operand then has a column for (query, even) and one for (query, odd), with P_b in one half of
// a register and zero in the other, so a column gathers its own dims.  N = 8 holds 4 queries this
// way (groups of up to 8 take two column tiles from the same decoded operands), and the scores' columns are
// doubled to match, so that P goes from accumulator to operand layout through two movmatrix.
// For fp32 the two columns of a query hold the upper and lower f16 of q, 22 bits together at no cost, and
// P_b goes in twice, its rounding error in f16 after it.
//
// Work, ring and joins: decode_segments.cuh (139 KB of copies in flight per SM with 16 warps at D = 128, 104 KB with 12).
// Filling the ring with four bulk copies a unit, waited for on an mbarrier, took 5 to 9% longer than with 16-byte
// cp.async (96 x 8192, 32/8 heads of 128: 168 us against 155).
//
// Measured (bf16, 32/8 heads): 96 x 8192, head_dim 128: 157 us, 5.4 TB/s (84% of the copy rate), 64% of the
// ALU pipe's cycles, which the conversions, masks and shifts of the scales take (fp32: 191 us); 32 x 8192, head_dim 256:
// 107 us, 5.3 TB/s; 96: 56 us, 3.8 TB/s (its scales are read byte by byte); 1 x 131072, head_dim 128: 35.5 us,
// of which 24 are the loop, the rest the start's dependent reads (lengths, table, pages) and the second launch.
// 12 warps of three stages at head_dim 128: 168 us where 16 of two take 155; a third stage at 64 gains nothing.
#include <type_traits>

#include "common.cuh"
#include "decode_segments.cuh"
#include "mxfp4.cuh"

namespace mi {

namespace {

constexpr int kQueries = 4;          // query heads of a column tile
constexpr float kLift = 12.f;       // p is held as 2^(x - m + kLift): f16 reaches 2^-37 of the largest p
constexpr float kLag = 3.f;         // m may be this far behind: p <= 2^15
constexpr float kExact = 0x1p20f;   // kLift - m is off by 2^-4 at most for m up to here
constexpr uint32_t kLowestRef = 0x20202020u;  // R_b - 255 then has a bit of 0xf8 set, like every far scale

// NB blocks of 32 per head, CT column tiles of 4 query heads, SPLIT: fp32.  One tile leaves the registers for
// 16 warps, two at D = 128 and fp32 for 12; past D = 128 shared memory holds the rings of 8 (and one tile).
template <int NB, bool SPLIT, int CT>
constexpr int kMxWarps = NB > 4 ? 8 : (CT == 1 || NB <= 2) && !SPLIT ? 16 : 12;
template <int NB, int CT, bool SPLIT>
struct MxCfg : SegCfg<NB * kMxBlock, kMxWarps<NB, SPLIT, CT>, 2, CT * kQueries, NB * kMxBytes, CT * NB * 512> {
  // Scale bytes are held four to a word, a word per 4 blocks of a key; at D = 64 a word has two keys'.
  static constexpr int kQuads = (NB + 3) / 4;
  static constexpr bool kBytes = NB != 2 && NB % 4 != 0;  // a key's bytes do not make words in memory
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
// Both halves of a times the low (HIGH: high) half of b.
template <bool HIGH>
__device__ __forceinline__ uint32_t mul_f16x2_half(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (HIGH)
    asm("{ .reg .b16 l, h; .reg .b32 x; mov.b32 {l, h}, %2; mov.b32 x, {h, h}; mul.rn.f16x2 %0, %1, x; }"
        : "=r"(r)
        : "r"(a), "r"(b));
  else
    asm("{ .reg .b16 l, h; .reg .b32 x; mov.b32 {l, h}, %2; mov.b32 x, {l, l}; mul.rn.f16x2 %0, %1, x; }"
        : "=r"(r)
        : "r"(a), "r"(b));
  return r;
}

// The codes of a group as MMA A fragments: its 2 NB matrices of 8 keys x 16 bytes lie one after the other.
// NB registers for keys 0-7 and 8-15 each.
template <int NB, bool TRANS>
__device__ __forceinline__ void load_codes(uint32_t base, int lane, uint32_t (&lo)[NB], uint32_t (&hi)[NB]) {
  const int mi = lane >> 3, rr = lane & 7;
  if constexpr (NB == 4) {
    const uint32_t addr = base + mi * kMxBlockBytes + rr * 16;
    if constexpr (TRANS) {
      ldsm4t(addr, lo[0], lo[1], lo[2], lo[3]);
      ldsm4t(addr + 128, hi[0], hi[1], hi[2], hi[3]);
    } else {
      ldsm4(addr, lo[0], lo[1], lo[2], lo[3]);
      ldsm4(addr + 128, hi[0], hi[1], hi[2], hi[3]);
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; b += 2) {
      uint32_t lo1, hi1;  // an odd NB's last block is read twice
      const uint32_t addr = base + b * kMxBlockBytes + (b + 1 < NB ? lane : lane & 15) * 16;
      if constexpr (TRANS)
        ldsm4t(addr, lo[b], hi[b], lo1, hi1);
      else
        ldsm4(addr, lo[b], hi[b], lo1, hi1);
      if (b + 1 < NB) lo[b + 1 < NB ? b + 1 : 0] = lo1, hi[b + 1 < NB ? b + 1 : 0] = hi1;
    }
  }
}

// 2^(e - 127) (1 + 2^-23) of byte b: the low bit makes the byte 255 a NaN, and all scores share the factor.
__device__ __forceinline__ float scale_of(uint32_t w, int b) {
  const uint32_t v = b == 0 ? w << 23 : b == 1 ? w << 15 : b == 2 ? w << 7 : w >> 1;
  return __uint_as_float((v & 0x7f800000u) | 1u);
}

__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(addr));
  return r;
}

// V's scales of a group, words of blocks 4i to 4i + 3: of keys 2t, 2t + 1 (w[i][0], w[i][1]) and 2t + 8, 2t + 9
// (w[i][2], w[i][3]); at D = 64 a key pair has one word.  Bytes of blocks that do not exist are kPadScale.
constexpr uint32_t kPadScale = kLowestRef & 255u;
template <int NB, int Q>
__device__ __forceinline__ void load_scales(uint32_t vbase, int t, uint32_t (&w)[Q][4]) {
  const uint32_t at = vbase + NB * kMxBlockBytes;
  if constexpr (NB == 4) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0][0]), "=r"(w[0][1]) : "r"(at + t * 8));
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0][2]), "=r"(w[0][3]) : "r"(at + t * 8 + 32));
  } else if constexpr (NB == 2) {
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0][0]) : "r"(at + t * 4));
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0][2]) : "r"(at + t * 4 + 16));
    w[0][1] = w[0][3] = 0;
  } else if constexpr (NB == 8) {
#pragma unroll
    for (int k = 0; k < 4; k += 2)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0][k]), "=r"(w[1][k]), "=r"(w[0][k + 1]), "=r"(w[1][k + 1])
                   : "r"(at + t * 16 + k * 32));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        w[i][k] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          w[i][k] |= (4 * i + b < NB ? lds8(at + (2 * t + (k & 1) + (k >> 1) * 8) * NB + 4 * i + b) : kPadScale) << (8 * b);
      }
  }
}

// A warp's state on a segment: 4 query heads to a column tile, lane (g, t) = (lane / 4, lane % 4).
template <typename T, int NB, int CT>
struct MxWarp {
  static constexpr bool kSplit = std::is_same<T, float>::value;
  using Elem_ = T;
  static constexpr int kSlack = 1;
  static constexpr bool kBulk = false;
  using C = MxCfg<NB, CT, kSplit>;
  static constexpr int D = C::D;
  static constexpr int kParts = kSplit ? 2 : 1;  // f16 parts of p
  static constexpr int Q = C::kQuads;
  uint32_t q;                 // shared address of this lane's B fragments of q (columns 2i and 2i + 1 both
                              // query i of the tile): 4 words per block, 512 bytes between blocks
  float xs[CT];               // log2-domain scale of query t
  float o[CT][NB][4];         // query t, dims 32b + 4g + 0 to 3, times 2^(R_b - 127)
  float m[CT], l[CT];         // query t; l: this lane's keys only
  uint32_t ref[Q];            // R_b, one byte per block
  uint32_t pick0, pick1;      // byte selectors: a pair's first (second) half to this lane's column, zeros
  int lane, g, t;

  __device__ __forceinline__ void setup(uint32_t query_smem) {
    lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    q = query_smem + lane * 16;
    pick0 = g & 1 ? 0x1044u : 0x4410u, pick1 = g & 1 ? 0x3244u : 0x4432u;
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < Q; ++i) ref[i] = kLowestRef;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
      for (int b = 0; b < NB; ++b) o[c][b][0] = o[c][b][1] = o[c][b][2] = o[c][b][3] = 0.f;
      m[c] = -INFINITY;
      l[c] = 0.f;
    }
  }

  // q of the segment's query heads (heads of them exist): this lane's elements ...
  static constexpr int kRaw = 8 * static_cast<int>(sizeof(T)) / 16;
  using Raw = uint4[CT][NB][kRaw];
  __device__ __forceinline__ void fetch_query(const T *query, int heads, Raw &raw) const {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int h = c * kQueries + (g >> 1);
#pragma unroll
      for (int i = 0; i < NB * kRaw; ++i) {
        uint4 &v = raw[c][i / kRaw][i % kRaw];
        v = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads) v = reinterpret_cast<const uint4 *>(query + h * D + i / kRaw * 32 + t * 8)[i % kRaw];
      }
    }
  }
  // ... as f16 fragments.
  __device__ __forceinline__ void set_query(const Raw &raw, float scale_log2) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float x[NB][8];
      uint32_t top = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if constexpr (kSplit) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 &v = raw[c][b][i];
            x[b][4 * i] = __uint_as_float(v.x), x[b][4 * i + 1] = __uint_as_float(v.y);
            x[b][4 * i + 2] = __uint_as_float(v.z), x[b][4 * i + 3] = __uint_as_float(v.w);
          }
        } else {
          float2 f[4];
          Vec16<T>::unpack(raw[c][b][0], f);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[b][2 * i] = f[i].x, x[b][2 * i + 1] = f[i].y;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[b][i]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(kAll, top, 1));
      top = max(top, __shfl_xor_sync(kAll, top, 2));
      int e = 14 - (static_cast<int>(top >> 23) - 127);  // largest element to [2^14, 2^15)
      if (top >= 0x7f800000u) e = 0;                     // not finite: as it is
      e = min(e, 126);
      const float f = exp2i(e);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[b][i] *= f;
          if (kSplit && (g & 1)) x[b][i] -= __half2float(__float2half_rn(x[b][i]));  // what the other column leaves
        }
        // read by this lane alone
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q + (c * NB + b) * 512),
                     "r"(pack_f16(x[b][0], x[b][1])), "r"(pack_f16(x[b][2], x[b][3])),
                     "r"(pack_f16(x[b][4], x[b][5])), "r"(pack_f16(x[b][6], x[b][7]))
                     : "memory");
      }
      xs[c] = __shfl_sync(kAll, exp2i(-e) * scale_log2, 8 * t);  // a lane of query t: g = 2t
    }
  }

  // Scores of a unit's 32 keys for query t: x[j][c][0], key g of group j; x[j][c][1], its key g + 8.
  // K's scale comes before xs, which takes q's lift back: one multiplication a score for that.
  __device__ __forceinline__ void scores(uint32_t kbase, float (&x)[2][CT][2]) const {
    constexpr int kWords = C::kBytes ? NB : Q;  // scales of a key: bytes of their own, or words of four
    uint32_t lo[2][NB], hi[2][NB], wl[2][kWords], wh[2][kWords];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t base = kbase + j * C::kGroup, at = base + NB * kMxBlockBytes + g * NB;
      load_codes<NB, false>(base, lane, lo[j], hi[j]);
      if constexpr (NB == 4) {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wl[j][0]) : "r"(at));
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wh[j][0]) : "r"(at + 8 * NB));
      } else if constexpr (NB == 2) {
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(wl[j][0]) : "r"(at));
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(wh[j][0]) : "r"(at + 8 * NB));
      } else if constexpr (NB == 8) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wl[j][0]), "=r"(wl[j][1]) : "r"(at));
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wh[j][0]), "=r"(wh[j][1]) : "r"(at + 8 * NB));
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) wl[j][b] = lds8(at + b), wh[j][b] = lds8(at + 8 * NB + b);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t f[CT][4];
#pragma unroll
      for (int c = 0; c < CT; ++c)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(f[c][0]), "=r"(f[c][1]), "=r"(f[c][2]), "=r"(f[c][3])
                     : "r"(q + (c * NB + b) * 512));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t a[4], e[4];
        mx_codes_to_f16(lo[j][b], a);
        mx_codes_to_f16(hi[j][b], e);
        const float fl = C::kBytes ? scale_of(wl[j][b % kWords], 0) : scale_of(wl[j][b / 4 % kWords], b % 4);
        const float fh = C::kBytes ? scale_of(wh[j][b % kWords], 0) : scale_of(wh[j][b / 4 % kWords], b % 4);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          float d[4];
          mma_f16_zero(d, a[0], e[0], a[1], e[1], f[c][0], f[c][1]);
          mma_f16(d, a[2], e[2], a[3], e[3], f[c][2], f[c][3]);
          if constexpr (kSplit) d[0] += d[1], d[2] += d[3];
          x[j][c][0] = b == 0 ? d[0] * fl : fmaf(d[0], fl, x[j][c][0]);
          x[j][c][1] = b == 0 ? d[2] * fh : fmaf(d[2], fh, x[j][c][1]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < CT; ++c) x[j][c][0] *= xs[c], x[j][c][1] *= xs[c];
  }

  // d * scale * x, the scales first: their product is in the range of the term itself where d is not far from q's
  // lift (a d of zero, or of q's smallest elements, leaves them apart).
  __device__ __forceinline__ static float far_term(float d, float scale, float x) {
    const float both = scale * x;
    return fabsf(both) <= 0x1p127f ? d * both : d * x * scale;
  }

  // As scores() where its order of the factors leaves fp32's range though the score may not: q is up to 2^15 here,
  // so keys of 2^105 do.
  // Rolled up: unrolled like the other it costs 16 bytes of spills at D = 128.
  __device__ __forceinline__ void scores_far(uint32_t kbase, float (&x)[2][CT][2]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t base = kbase + j * C::kGroup, at = base + NB * kMxBlockBytes + g * NB;
#pragma unroll
      for (int c = 0; c < CT; ++c) x[j][c][0] = x[j][c][1] = 0.f;
#pragma unroll 1
      for (int b = 0; b < NB; ++b) {
        uint32_t lo, hi, again[2], a[4], e[4];
        ldsm4(base + b * kMxBlockBytes + (lane & 15) * 16, lo, hi, again[0], again[1]);
        mx_codes_to_f16(lo, a);
        mx_codes_to_f16(hi, e);
        const float fl = scale_of(lds8(at + b), 0), fh = scale_of(lds8(at + 8 * NB + b), 0);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          uint32_t f[4];
          float d[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
                       : "r"(q + (c * NB + b) * 512));
          mma_f16_zero(d, a[0], e[0], a[1], e[1], f[0], f[1]);
          mma_f16(d, a[2], e[2], a[3], e[3], f[2], f[3]);
          if constexpr (kSplit) d[0] += d[1], d[2] += d[3];
          x[j][c][0] += far_term(d[0], fl, xs[c]);
          x[j][c][1] += far_term(d[2], fh, xs[c]);
        }
      }
    }
  }

  // Scale bytes of keys that do not exist become `with`'s.
  __device__ __forceinline__ void mask_scales(uint32_t (&w)[Q][4], int valid, const uint32_t (&with)[Q]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (2 * t + (k & 1) + (k >> 1) * 8 < valid) continue;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        if constexpr (NB == 2)
          w[i][k & 2] = k & 1 ? (w[i][k & 2] & 0xffffu) | with[i] << 16 : (w[i][k & 2] & 0xffff0000u) | (with[i] & 0xffffu);
        else
          w[i][k] = with[i];
      }
    }
  }

  // How far below the reference each scale is, per byte: 0 to 7, or a bit of 0xf8 is set in the result.
  __device__ __forceinline__ uint32_t distances(const uint32_t (&w)[Q][4], uint32_t (&d)[Q][4]) const {
    if constexpr (NB == 2) {
      const uint32_t both = (ref[0] & 0xffffu) * 0x10001u;
      d[0][0] = both - w[0][0], d[0][2] = both - w[0][2];
      return (d[0][0] | d[0][2]) & 0xf8f8f8f8u;
    } else {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) d[i][k] = ref[i] - w[i][k];
        any |= d[i][0] | d[i][1] | d[i][2] | d[i][3];
      }
      return any & 0xf8f8f8f8u;
    }
  }

  // O += P_b V of a group.  d: distances per byte, 0 to 7, or 15 for no contribution (2^-15 has the f16
  // exponent 0: zero); p[part][c][k]: p of keys 2t, 2t + 1, 2t + 8, 2t + 9 in the half of this lane's
  // column, zero in the other (fp32: its upper f16, then its lower).  FAR: the products are `back` times what d says.
  template <bool FAR>
  __device__ __forceinline__ void values(uint32_t vbase, const uint32_t (&d)[Q][4], const uint32_t (&p)[kParts][CT][4],
                                         float back = 1.f) {
    uint32_t lo[NB], hi[NB];
    load_codes<NB, true>(vbase, lane, lo, hi);
    // f16 2^-d, two to a word: bytes 0 and 2 of d's word k, then bytes 1 and 3
    uint32_t even[Q][4], odd[Q][4];
#pragma unroll
    for (int i = 0; i < Q; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (NB == 2 && (k & 1)) continue;
        even[i][k] = 0x3c003c00u - (d[i][k] & 0x00ff00ffu) * 1024u;
        odd[i][k] = 0x3c003c00u - (d[i][k] & 0xff00ff00u) * 4u;
      }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t a[4], e[4];
      mx_codes_to_f16(lo[b], a);
      mx_codes_to_f16(hi[b], e);
#pragma unroll
      for (int part = 0; part < kParts * CT; ++part) {
        const int c = part / kParts, half = part % kParts;
        uint32_t s[4];  // p times the scale of V's block b
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t pk = p[half][c][k];
          if constexpr (NB == 2) {
            const uint32_t f = b & 1 ? odd[0][k & 2] : even[0][k & 2];
            s[k] = k & 1 ? mul_f16x2_half<true>(pk, f) : mul_f16x2_half<false>(pk, f);
          } else {
            const uint32_t f = b & 1 ? odd[b / 4][k] : even[b / 4][k];
            s[k] = b % 4 < 2 ? mul_f16x2_half<false>(pk, f) : mul_f16x2_half<true>(pk, f);
          }
        }
        if constexpr (FAR) {
          float r[4];
          mma_f16_zero(r, a[0], a[1], a[2], a[3], s[0], s[1]);
          mma_f16(r, e[0], e[1], e[2], e[3], s[2], s[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[c][b][i] = fmaf(r[i], back, o[c][b][i]);
        } else {
          mma_f16(o[c][b], a[0], a[1], a[2], a[3], s[0], s[1]);
          mma_f16(o[c][b], e[0], e[1], e[2], e[3], s[2], s[3]);
        }
      }
    }
  }

  // The largest byte of each block over the group's keys, from this lane's four.
  __device__ __forceinline__ static uint32_t over_keys(const uint32_t (&w)[4]) {
    uint32_t top = __vmaxu4(__vmaxu4(w[0], w[1]), __vmaxu4(w[2], w[3]));
    if constexpr (NB == 2) top = __vmaxu4(top, top >> 16) & 0xffffu;
    top = __vmaxu4(top, __shfl_xor_sync(kAll, top, 1));
    return __vmaxu4(top, __shfl_xor_sync(kAll, top, 2));
  }

  // As values() for scales that the window of 8 binades does not hold: raise R_b where a scale is above
  // it, then take the keys window by window.
  __device__ __forceinline__ void values_far(uint32_t vbase, const uint32_t (&p)[kParts][CT][4], int valid) {
    uint32_t w[Q][4], some[Q][4], bad[Q], any_bad = 0, deepest = 0;  // some: all ones where there is a scale
    const uint32_t none[Q] = {};
    load_scales<NB>(vbase, t, w);
    mask_scales(w, valid, none);
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      uint32_t nan[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        nan[k] = __vcmpeq4(w[i][k], 0xffffffffu);
        w[i][k] &= ~nan[k];
      }
      bad[i] = over_keys(nan);
      any_bad |= bad[i];
      const uint32_t top = over_keys(w[i]);
      const uint32_t above = __vcmpgtu4(top, ref[i]);
      const uint32_t next = (ref[i] & ~above) | (__vminu4(__vaddus4(top, 0x02020202u), 0xfefefefeu) & above);
#pragma unroll
      for (int b = 4 * i; b < NB && b < 4 * i + 4; ++b) {
        const float f = exp2i(static_cast<int>((ref[i] >> (8 * (b % 4))) & 255u) -
                              static_cast<int>((next >> (8 * (b % 4))) & 255u));
#pragma unroll
        for (int u = 0; u < CT * 4; ++u) o[u / 4][b][u % 4] *= f;
      }
      ref[i] = next;
      const uint32_t all = NB == 2 ? (ref[i] & 0xffffu) * 0x10001u : ref[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        some[i][k] = __vcmpne4(w[i][k], 0u);
        w[i][k] = (all - w[i][k]) & some[i][k];  // no byte is above the reference now
      }
      deepest = __vmaxu4(deepest, over_keys(w[i]));
    }
    deepest = __vmaxu4(deepest, deepest >> 16);
    deepest = max(deepest & 255u, (deepest >> 8) & 255u);
#pragma unroll 1
    for (uint32_t window = 0; window <= deepest / 8; ++window) {
      uint32_t d[Q][4];
#pragma unroll
      for (int i = 0; i < Q; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t in = __vcmpeq4((w[i][k] >> 3) & 0x1f1f1f1fu, window * 0x01010101u) & some[i][k];
          d[i][k] = (w[i][k] & 0x07070707u & in) | (0x0f0f0f0fu & ~in);
        }
      values<true>(vbase, d, p, exp2i(-8 * static_cast<int>(window)));
    }
    if (any_bad) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (bad[b / 4] >> (8 * (b % 4)) & 255u)
#pragma unroll
          for (int i = 0; i < CT * 4; ++i) o[i / 4][b][i % 4] = __uint_as_float(0x7fffffffu);
    }
  }

  // One unit: K of its two groups at `base`, then V of both; `valid0` and `valid1` of their 16 keys exist; `special`:
  // that may be fewer than 16, or it is the `first` that the state meets.
  __device__ __forceinline__ void process(uint32_t base, bool special, int valid0, int valid1, bool first) {
    const uint32_t vbase = base + 2 * C::kGroup;
    float x[2][CT][2];
    scores(base, x);
    uint32_t w[2][Q][4];
    load_scales<NB>(vbase, t, w[0]);
    load_scales<NB>(vbase + C::kGroup, t, w[1]);
    bool far_scores = false;  // a score may not be finite because of how it was multiplied
#pragma unroll
    for (int c = 0; c < CT; ++c)
      far_scores |= !(fabsf((x[0][c][0] + x[0][c][1]) + (x[1][c][0] + x[1][c][1])) <= 0x1p126f);
    if (__any_sync(kAll, far_scores)) scores_far(base, x);
    if (special) {  // uniform
      if (first) {  // R_b starts at the largest scale here and two binades of room
        const uint32_t none[Q] = {};
        mask_scales(w[0], valid0, none);
        mask_scales(w[1], valid1, none);
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const uint32_t top = __vmaxu4(over_keys(w[0][i]), over_keys(w[1][i]));
          ref[i] = __vmaxu4(__vminu4(__vaddus4(top, 0x02020202u), 0xfefefefeu), kLowestRef);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (g >= (j ? valid1 : valid0)) x[j][c][0] = -INFINITY;
          if (g + 8 >= (j ? valid1 : valid0)) x[j][c][1] = -INFINITY;
        }
        mask_scales(w[j], j ? valid1 : valid0, ref);  // whatever they are: their p is zero
      }
    }
    // m follows the largest score, up to kLag binades behind it (by the difference: m + kLag may round to m + 4 from 2^24 on)
    float top[CT];
    bool behind = false;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      top[c] = fmaxf(fmaxf(x[0][c][0], x[0][c][1]), fmaxf(x[1][c][0], x[1][c][1]));
      behind |= top[c] - m[c] > kLag;
    }
    if (__any_sync(kAll, behind)) {
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        float mx = top[c];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, off));
        if (mx > m[c]) {  // the lanes of a query agree
          const float f = m[c] == -INFINITY ? 0.f : fast_exp2(m[c] - mx);
#pragma unroll
          for (int i = 0; i < NB * 4; ++i) o[c][i / 4][i % 4] *= f;
          l[c] *= f;
          m[c] = mx;
        }
      }
    }
    uint32_t p[2][kParts][CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float lift = kLift - m[c];
      if (fabsf(m[c]) > kExact) {  // which m would round away: m goes at once
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i / 2][c][i % 2] -= m[c];
        lift = kLift;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float p0 = fast_exp2(x[j][c][0] + lift), p1 = fast_exp2(x[j][c][1] + lift);
        l[c] += p0 + p1;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          // rows (keys) x columns (each query twice), transposed: keys 2t and 2t + 1 of query g / 2
          const uint32_t k0 = movm(pack_f16(p0, p0)), k8 = movm(pack_f16(p1, p1));
          p[j][part][c][0] = __byte_perm(k0, 0, pick0), p[j][part][c][1] = __byte_perm(k0, 0, pick1);
          p[j][part][c][2] = __byte_perm(k8, 0, pick0), p[j][part][c][3] = __byte_perm(k8, 0, pick1);
          if (part + 1 < kParts) p0 -= __half2float(__float2half_rn(p0)), p1 -= __half2float(__float2half_rn(p1));
        }
      }
    }
    uint32_t d[2][Q][4];
    const uint32_t far = distances(w[0], d[0]) | distances(w[1], d[1]);
    if (__any_sync(kAll, far != 0)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) values_far(vbase + j * C::kGroup, p[j], j ? valid1 : valid0);
    } else {
      values<false>(vbase, d[0], p[0]);
      values<false>(vbase + C::kGroup, d[1], p[1]);
    }
  }

  // Sum l over the keys of the lanes.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[c] += __shfl_xor_sync(kAll, l[c], off);
  }

  // The mean of V over the keys seen: o is divided by l, which holds the lift of p as o does, before the scale comes
  // back, so that the result is in range where V is.
  __device__ __forceinline__ float inverse(int c) const { return l[c] == 0.f ? 0.f : __fdividef(1.f, l[c]); }
  __device__ __forceinline__ float scale_back(int b) const {
    return exp2i(static_cast<int>((ref[b / 4] >> (8 * (b % 4))) & 255u) - 127);
  }

  __device__ __forceinline__ void write_out(T *out, int heads) const {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if (c * kQueries + t >= heads) continue;
      const float inv = inverse(c);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        using V = typename std::conditional<kSplit, uint4, uint2>::type;
        const float f = scale_back(b);
        V v;
        T *e = reinterpret_cast<T *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = Elem<T>::from_float(o[c][b][i] * inv * f);
        *reinterpret_cast<V *>(out + (c * kQueries + t) * D + b * 32 + g * 4) = v;
      }
    }
  }

  __device__ __forceinline__ void write_state(float *st, int heads) const {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int h = c * kQueries + t;
      if (h >= heads) continue;
      const float inv = inverse(c);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float f = scale_back(b);
        *reinterpret_cast<float4 *>(st + h * D + b * 32 + g * 4) = make_float4(
            o[c][b][0] * inv * f, o[c][b][1] * inv * f, o[c][b][2] * inv * f, o[c][b][3] * inv * f);
      }
      if (g == 0) {
        st[C::kHeads * D + h] = m[c];
        st[C::kHeads * D + C::kHeads + h] = l[c];
      }
    }
  }
};

template <typename T, int NB, int CT>
__global__ void __launch_bounds__(MxCfg<NB, CT, std::is_same<T, float>::value>::kWarps * 32, 1)
    mxfp4_decode_mma_kernel(const CodedDecodeParams p, const SegPlan plan) {
  decode_segments<MxWarp<T, NB, CT>>(p, plan);
}

template <typename T, int NB, int CT>
__global__ void __launch_bounds__(kJoinLanes * kJoinWays)
    mxfp4_decode_mma_join_kernel(const CodedDecodeParams p, const SegPlan plan) {
  join_segments<MxWarp<T, NB, CT>>(p, plan);
}

template <typename T, int NB, int CT>
cudaError_t launch_mma(const CodedDecodeParams &p, int tiles, bool join, int ctas, cudaStream_t stream) {
  return launch_segments<MxWarp<T, NB, CT>>(mxfp4_decode_mma_kernel<T, NB, CT>, mxfp4_decode_mma_join_kernel<T, NB, CT>, p,
                                            tiles, join, ctas, stream);
}

// Column tiles of a segment (two rings' worth of sums do not fit past D = 128), and segments of a kv head.
int mma_columns(int num_q_heads, int num_kv_heads, int head_dim) {
  return num_q_heads / num_kv_heads <= kQueries || head_dim > 128 ? 1 : 2;
}
int mma_tiles(int num_q_heads, int num_kv_heads, int head_dim) {
  const int heads = kQueries * mma_columns(num_q_heads, num_kv_heads, head_dim);
  return (num_q_heads / num_kv_heads + heads - 1) / heads;
}

bool mma_joins(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t capacity, int sms) {
  const int64_t segments = num_seqs * num_kv_heads * mma_tiles(num_q_heads, num_kv_heads, head_dim);
  // the fewest warps of a CTA, at a slack of one unit each
  return segments_join(segments, capacity, head_dim > 128 ? MxCfg<8, 1, true>::kWarps : MxCfg<4, 2, true>::kWarps, sms);
}

template <typename T>
cudaError_t launch_mma_t(const CodedDecodeParams &p, int tiles, int columns, bool join, int ctas, cudaStream_t stream) {
  switch (p.head_dim / kMxBlock * 2 + columns) {
    case 3: return launch_mma<T, 1, 1>(p, tiles, join, ctas, stream);
    case 4: return launch_mma<T, 1, 2>(p, tiles, join, ctas, stream);
    case 5: return launch_mma<T, 2, 1>(p, tiles, join, ctas, stream);
    case 6: return launch_mma<T, 2, 2>(p, tiles, join, ctas, stream);
    case 7: return launch_mma<T, 3, 1>(p, tiles, join, ctas, stream);
    case 8: return launch_mma<T, 3, 2>(p, tiles, join, ctas, stream);
    case 9: return launch_mma<T, 4, 1>(p, tiles, join, ctas, stream);
    case 10: return launch_mma<T, 4, 2>(p, tiles, join, ctas, stream);
    case 11: return launch_mma<T, 5, 1>(p, tiles, join, ctas, stream);
    case 13: return launch_mma<T, 6, 1>(p, tiles, join, ctas, stream);
    case 15: return launch_mma<T, 7, 1>(p, tiles, join, ctas, stream);
    case 17: return launch_mma<T, 8, 1>(p, tiles, join, ctas, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

bool mxfp4_decode_supported(int num_q_heads, int num_kv_heads, int head_dim, int64_t num_blocks, int block_size,
                            int64_t capacity) {
  return segments_supported(static_cast<int64_t>(num_kv_heads) * mma_tiles(num_q_heads, num_kv_heads, head_dim),
                            num_kv_heads, num_blocks, block_size, capacity);
}

size_t mxfp4_decode_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t capacity,
                              int sms) {
  sms = segment_ctas(sms);
  if (!mma_joins(num_seqs, num_q_heads, num_kv_heads, head_dim, capacity, sms)) return 0;
  return segment_workspace(kQueries * mma_columns(num_q_heads, num_kv_heads, head_dim), head_dim, sms);
}

cudaError_t launch_mxfp4_decode(const CodedDecodeParams &p, int dtype, cudaStream_t stream) {
  const int tiles = mma_tiles(p.num_q_heads, p.num_kv_heads, p.head_dim);
  const int columns = mma_columns(p.num_q_heads, p.num_kv_heads, p.head_dim);
  const int sms = segment_ctas(sm_count_current());
  const bool join = mma_joins(p.num_seqs, p.num_q_heads, p.num_kv_heads, p.head_dim, p.bt_stride * p.block_size, sms);
  return launch_segment_slices(p, tiles, dtype, [&](const CodedDecodeParams &q) {
    return dtype == MI_DTYPE_BFLOAT16 ? launch_mma_t<__nv_bfloat16>(q, tiles, columns, join, sms, stream)
           : dtype == MI_DTYPE_FLOAT16  ? launch_mma_t<__half>(q, tiles, columns, join, sms, stream)
                                        : launch_mma_t<float>(q, tiles, columns, join, sms, stream);
  });
}

}  // namespace mi
