// Paged decode over the 4-bit cache on the warp-level tensor cores (bf16 and
// fp16, head_dim 64 or 128, any GQA group; other shapes: decode_mxfp4.cu).
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
//     8 binades, so no spread of scales loses more;
//   - q is multiplied by a power of two that puts its largest element into
//     [2^14, 2^15) and converted to f16 (exact for bf16 down to 2^-28 of that element).
// Fragments need no transposition of codes: an ldmatrix of 8 keys x 16 bytes gives
// each lane 8 consecutive codes of its key (K, dims in any order as long as q
// follows it), and the transposed one gives 4 codes of two neighbouring keys, which two
// bit-selects interleave to key pairs (V).  P goes from accumulator to operand
// layout through two movmatrix.
//
// Work: the groups of 16 keys of all (sequence, kv head, 8 query heads)
// segments, in that order, are one list that is cut into equal ranges, one per
// warp (16 warps to a CTA, one CTA to an SM), so ragged batches and single long
// sequences load every SM alike.  A warp streams its range through a ring of bulk copies
// (one of K and one of V per group; 4 stages, 139 KB in flight per SM at D = 128)
// that runs across segment borders.  Segments that lie within one
// warp's range are written at once; the parts of others are joined in shared
// memory, and those that cross CTAs by a second launch, whose order is fixed.
// When every segment fits a CTA at hardly more work per warp, each CTA takes one
// segment and the second launch has nothing to do.
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "params.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 16;
constexpr int kStages = 4;
constexpr int kCols = 8;            // query heads of a segment: the MMA's N
constexpr int kMaxSeqs = 2048;      // sequences of one launch (prefix sums in shared memory)
constexpr float kLift = 12.f;       // p is held as 2^(x - m + kLift): f16 reaches 2^-37 of the largest p
constexpr float kLag = 3.f;         // m may be this far behind: p <= 2^15
constexpr int kAlignedSlack = 2;    // groups per warp that keeping a segment in one CTA may cost

template <int NB>
struct MxCfg {
  static constexpr int D = NB * kMxBlock;
  static constexpr int kGroup = NB * kMxBytes;  // bytes of one group of one operand
  static constexpr int kStage = 2 * kGroup;
  static constexpr int kRing = kStages * kStage;  // per warp
  static constexpr int kState = kCols * (D + 2);  // floats: acc [8][D], m [8], l [8]
  static constexpr int kSmemRing = kWarps * kRing;
  static constexpr int kSmemHeads = kWarps * kState * 4;  // parts that end before their warp's range does
  static constexpr int kSmemBars = kWarps * kStages * 8;
  static constexpr int kSmemPrefix = (kMaxSeqs + 1) * 4;
  static constexpr int kSmemMisc = 4 * kWarps * 4 + 8 * kWarps + 64;
  static constexpr int kSmem = kSmemRing + kSmemHeads + kSmemBars + kSmemPrefix + kSmemMisc;
  static_assert(kState * 4 <= kRing, "a warp's last part goes into its own ring");
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// What a CTA leaves in the workspace beside its states: the segment of its first
// part if that began in an earlier CTA, whether it ends here, and the segment
// of its last part if that began here and goes on (-1: none).
struct MxMeta {
  int32_t head, head_ends, tail, pad;
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
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^e for any e, through two factors where one has no normal exponent.
__device__ __forceinline__ float exp2i(int e) {
  const int a = max(-126, min(127, e)), b = max(-126, min(127, e - a));
  return __uint_as_float(static_cast<uint32_t>(a + 127) << 23) * __uint_as_float(static_cast<uint32_t>(b + 127) << 23);
}

// The codes of a group as MMA A fragments.  NB registers for keys 0-7 and 8-15 each.
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
    const uint32_t addr = base + (mi >> 1) * kMxBlockBytes + (mi & 1) * 128 + rr * 16;
    if constexpr (TRANS)
      ldsm4t(addr, lo[0], hi[0], lo[1], hi[1]);
    else
      ldsm4(addr, lo[0], hi[0], lo[1], hi[1]);
  }
}

// Four codes of two keys (a: low 16 bits, b: high 16 bits) as f16 pairs (a_i, b_i).
__device__ __forceinline__ void key_pairs(uint32_t v, uint32_t (&e)[4]) {
  // bytes 2, 3 of x: (a1, b1), (a3, b3); of y: (a0, b0), (a2, b2)
  const uint32_t x = (v & 0xf0f0f0f0u) | ((v << 12) & 0x0f0f0f0fu);
  const uint32_t y = ((v << 4) & 0xf0f0f0f0u) | ((v << 16) & 0x0f0f0f0fu);
  asm("{ .reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %5;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b3; }"
      : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3])
      : "r"(x), "r"(y));
}

// One query head's state of a segment part, laid out [8][D] acc, [8] m, [8] l.
template <typename T, int NB>
struct MxWarp {
  using C = MxCfg<NB>;
  static constexpr int D = C::D;
  uint32_t q[NB * 2][2];  // B fragments of q
  float xs[2];            // log2-domain scale of queries 2t, 2t + 1
  float o[NB * 2][4];     // tile 2b + j: dims 32b + 4g + 2j (+ 1: [2], [3]), queries 2t, 2t + 1
  float m[2], l[2];
  uint32_t ref;           // R_b, one byte per block
  int lane, g, t;

  __device__ __forceinline__ void reset() {
    ref = 0x20202020u;  // the lowest reference: a byte of 255 is then never mistaken for a near one
#pragma unroll
    for (int i = 0; i < NB * 2; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }

  // Row `g` of the tile's query heads (heads of them exist).
  __device__ __forceinline__ void load_query(const T *query, int heads, float scale_log2) {
    float x[NB][8];
    uint32_t top = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (g < heads) v = *reinterpret_cast<const uint4 *>(query + g * D + b * 32 + t * 8);
      float2 f[4];
      Vec16<T>::unpack(v, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[b][2 * i] = f[i].x, x[b][2 * i + 1] = f[i].y;
        top = max(top, max(__float_as_uint(f[i].x) & 0x7fffffffu, __float_as_uint(f[i].y) & 0x7fffffffu));
      }
    }
    top = max(top, __shfl_xor_sync(kAll, top, 1));
    top = max(top, __shfl_xor_sync(kAll, top, 2));
    int e = 14 - (static_cast<int>(top >> 23) - 127);  // largest element to [2^14, 2^15)
    if (top >= 0x7f800000u) e = 0;                     // not finite: as it is
    e = min(e, 126);
    const float f = exp2i(e);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      q[2 * b][0] = pack_f16(x[b][0] * f, x[b][1] * f);
      q[2 * b][1] = pack_f16(x[b][2] * f, x[b][3] * f);
      q[2 * b + 1][0] = pack_f16(x[b][4] * f, x[b][5] * f);
      q[2 * b + 1][1] = pack_f16(x[b][6] * f, x[b][7] * f);
    }
    const float back = exp2i(-e) * scale_log2;
    xs[0] = __shfl_sync(kAll, back, 8 * t);  // lane of query 2t: g = 2t
    xs[1] = __shfl_sync(kAll, back, 8 * t + 4);
  }

  // P_b of this lane's keys times V's block b into `d0`, `d1` (rows j = 0, 1).
  __device__ __forceinline__ static void value_block(uint32_t lo, uint32_t hi, uint32_t p0, uint32_t p1,
                                                     float (&d0)[4], float (&d1)[4]) {
    uint32_t a[4], c[4];
    key_pairs(lo, a);
    key_pairs(hi, c);
    mma_f16(d0, a[0], a[1], c[0], c[1], p0, p1);
    mma_f16(d1, a[2], a[3], c[2], c[3], p0, p1);
  }

  // Scale byte of key pair word(s), block b, key `which` (0, 1) of the pair.
  __device__ __forceinline__ static uint32_t byte_of(const uint32_t (&w)[2], int b, int which) {
    if constexpr (NB == 4)
      return (w[which] >> (8 * b)) & 255u;
    else
      return (w[0] >> (16 * which + 8 * b)) & 255u;
  }

  // Scales that the window of 8 binades does not hold: raise R_b where a scale is above it,
  // then take the keys window by window.  `pp`: p of keys (2t, 2t+1) and (2t+8, 2t+9) of query g.
  __device__ __forceinline__ void value_slow(uint32_t vcodes, const uint32_t (&w0)[2], const uint32_t (&w1)[2],
                                          uint32_t pp0, uint32_t pp1) {
    int deepest = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      int top = 0, low = 255;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = byte_of(k < 2 ? w0 : w1, b, k & 1);
        if (s >= 1 && s <= 254) top = max(top, s), low = min(low, s);
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        top = max(top, __shfl_xor_sync(kAll, top, off));
        low = min(low, __shfl_xor_sync(kAll, low, off));
      }
      int r = (ref >> (8 * b)) & 255;
      if (top > r) {
        const int next = min(top + 2, 254);
        const float f = exp2i(r - next);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[2 * b + j][i] *= f;
        ref = (ref & ~(255u << (8 * b))) | (static_cast<uint32_t>(next) << (8 * b));
        r = next;
      }
      if (low < 255) deepest = max(deepest, r - low);
    }
    uint32_t lo[NB], hi[NB];
    load_codes<NB, true>(vcodes, lane, lo, hi);
#pragma unroll 1
    for (int window = 0; window <= deepest / 8; ++window) {
      const float back = exp2i(-8 * window);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int r = (ref >> (8 * b)) & 255;
        uint32_t f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int s = byte_of(k < 2 ? w0 : w1, b, k & 1), d = r - s;
          f[k] = s >= 1 && s <= 254 && (d >> 3) == window ? 0x3c00u - ((d & 7) << 10) : 0u;
          if (s == 255 && window == 0) f[k] = 0x7e00u;
        }
        float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
        value_block(lo[b], hi[b], mul_f16x2(pp0, f[0] | f[1] << 16), mul_f16x2(pp1, f[2] | f[3] << 16), d0, d1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[2 * b][i] = fmaf(d0[i], back, o[2 * b][i]);
          o[2 * b + 1][i] = fmaf(d1[i], back, o[2 * b + 1][i]);
        }
      }
    }
  }

  // One group: `kbase`, `vbase` its K and V bytes in shared memory, `valid` of its 16 keys exist.
  __device__ __forceinline__ void process(uint32_t kbase, uint32_t vbase, int valid) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};  // (key g, queries 2t, 2t + 1), (key g + 8, ...)
    {
      uint32_t lo[NB], hi[NB], wl, wh;
      load_codes<NB, false>(kbase, lane, lo, hi);
      if constexpr (NB == 4) {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wl) : "r"(kbase + NB * kMxBlockBytes + g * 4));
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wh) : "r"(kbase + NB * kMxBlockBytes + g * 4 + 32));
      } else {
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(wl) : "r"(kbase + NB * kMxBlockBytes + g * 2));
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(wh) : "r"(kbase + NB * kMxBlockBytes + g * 2 + 16));
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t a[4], c[4];
        mx_codes_to_f16(lo[b], a);
        mx_codes_to_f16(hi[b], c);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma_f16(d, a[0], c[0], a[1], c[1], q[2 * b][0], q[2 * b][1]);
        mma_f16(d, a[2], c[2], a[3], c[3], q[2 * b + 1][0], q[2 * b + 1][1]);
        // 2^(e - 127) (1 + 2^-23): the low bit makes the byte 255 a NaN, and all scores share the factor
        const float fl = __uint_as_float((((wl >> (8 * b)) & 255u) << 23) | 1u);
        const float fh = __uint_as_float((((wh >> (8 * b)) & 255u) << 23) | 1u);
        x[0] = fmaf(d[0], fl, x[0]);
        x[1] = fmaf(d[1], fl, x[1]);
        x[2] = fmaf(d[2], fh, x[2]);
        x[3] = fmaf(d[3], fh, x[3]);
      }
    }
    // V's scales: words of keys 2t, 2t + 1 and 2t + 8, 2t + 9
    uint32_t w0[2], w1[2];
    if constexpr (NB == 4) {
      asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w0[0]), "=r"(w0[1]) : "r"(vbase + NB * kMxBlockBytes + t * 8));
      asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                   : "=r"(w1[0]), "=r"(w1[1])
                   : "r"(vbase + NB * kMxBlockBytes + t * 8 + 32));
    } else {
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w0[0]) : "r"(vbase + NB * kMxBlockBytes + t * 4));
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w1[0]) : "r"(vbase + NB * kMxBlockBytes + t * 4 + 16));
      w0[1] = w1[1] = 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= xs[i & 1];
    if (valid < kMxGroup) {  // uniform: the last group of a sequence
      if (g >= valid) x[0] = x[1] = -INFINITY;
      if (g + 8 >= valid) x[2] = x[3] = -INFINITY;
      // stale scales of keys that do not exist become the reference (their p is zero)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (2 * t + (k & 1) + (k >> 1) * 8 < valid) continue;
        uint32_t(&w)[2] = k < 2 ? w0 : w1;
        if constexpr (NB == 4)
          w[k & 1] = ref;
        else
          w[0] = k & 1 ? (w[0] & 0xffffu) | ref << 16 : (w[0] & 0xffff0000u) | (ref & 0xffffu);
      }
    }
    const bool behind = fmaxf(x[0], x[2]) > m[0] + kLag || fmaxf(x[1], x[3]) > m[1] + kLag;
    if (__any_sync(kAll, behind)) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = fmaxf(x[c], x[c + 2]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, off));
        if (mx > m[c]) {  // the lanes of a query agree
          const float f = m[c] == -INFINITY ? 0.f : fast_exp2(m[c] - mx);
#pragma unroll
          for (int i = 0; i < NB * 2; ++i) o[i][c] *= f, o[i][c + 2] *= f;
          l[c] *= f;
          m[c] = mx;
        }
      }
    }
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = fast_exp2(x[i] - m[i & 1] + kLift);
    l[0] += p[0] + p[2];
    l[1] += p[1] + p[3];
    const uint32_t pp0 = movm(pack_f16(p[0], p[1])), pp1 = movm(pack_f16(p[2], p[3]));

    // how far below the reference each scale is, per byte
    uint32_t d0[2], d1[2], bad;
    if constexpr (NB == 4) {
#pragma unroll
      for (int k = 0; k < 2; ++k) d0[k] = ref - w0[k], d1[k] = ref - w1[k];
      bad = (d0[0] | d0[1] | d1[0] | d1[1]) & 0xf8f8f8f8u;
    } else {
      const uint32_t both = (ref & 0xffffu) * 0x10001u;
      d0[0] = both - w0[0], d1[0] = both - w1[0];
      bad = (d0[0] | d1[0]) & 0xf8f8f8f8u;
    }
    if (__any_sync(kAll, bad != 0)) {
      value_slow(vbase, w0, w1, pp0, pp1);
    } else {
      uint32_t lo[NB], hi[NB];
      load_codes<NB, true>(vbase, lane, lo, hi);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t z0, z1;  // d of the pair's keys in bits 8-11 and 24-27
        if constexpr (NB == 4) {
          z0 = __byte_perm(d0[0], d0[1], b << 4 | (b + 4) << 12);
          z1 = __byte_perm(d1[0], d1[1], b << 4 | (b + 4) << 12);
        } else {
          z0 = __byte_perm(d0[0], 0, b << 4 | (b + 2) << 12);
          z1 = __byte_perm(d1[0], 0, b << 4 | (b + 2) << 12);
        }
        const uint32_t f0 = 0x3c003c00u - ((z0 & 0x07000700u) << 2), f1 = 0x3c003c00u - ((z1 & 0x07000700u) << 2);
        value_block(lo[b], hi[b], mul_f16x2(pp0, f0), mul_f16x2(pp1, f1), o[2 * b], o[2 * b + 1]);
      }
    }
  }

  // Sum l over the keys of the lanes, bring o to its true scale.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[c] += __shfl_xor_sync(kAll, l[c], off);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float f = exp2i(static_cast<int>((ref >> (8 * b)) & 255u) - 127);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[2 * b][i] *= f, o[2 * b + 1][i] *= f;
    }
  }

  __device__ __forceinline__ void write_out(T *out, int heads) const {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (2 * t + c >= heads) continue;
      const float inv = l[c] == 0.f ? 0.f : 1.f / l[c];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint2 v;
        T *e = reinterpret_cast<T *>(&v);
        e[0] = Elem<T>::from_float(o[2 * b][c] * inv);
        e[1] = Elem<T>::from_float(o[2 * b][c + 2] * inv);
        e[2] = Elem<T>::from_float(o[2 * b + 1][c] * inv);
        e[3] = Elem<T>::from_float(o[2 * b + 1][c + 2] * inv);
        *reinterpret_cast<uint2 *>(out + (2 * t + c) * D + b * 32 + g * 4) = v;
      }
    }
  }

  __device__ __forceinline__ void write_state(float *st, int heads) const {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (2 * t + c >= heads) continue;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        *reinterpret_cast<float4 *>(st + (2 * t + c) * D + b * 32 + g * 4) =
            make_float4(o[2 * b][c], o[2 * b][c + 2], o[2 * b + 1][c], o[2 * b + 1][c + 2]);
      if (g == 0) {
        st[kCols * D + 2 * t + c] = m[c];
        st[kCols * D + kCols + 2 * t + c] = l[c];
      }
    }
  }
};

// exp2(m - M) of a part: 0 for one without a key, 1 where both are -inf or NaN (l carries the NaN).
__device__ __forceinline__ float part_factor(float m, float l, float M) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return fast_exp2(m - M);
}

template <typename T, int NB>
__global__ void __launch_bounds__(kWarps * 32, 1) mxfp4_decode_mma_kernel(const MxDecodeParams p, int tiles) {
  using C = MxCfg<NB>;
  constexpr int D = C::D;
  extern __shared__ __align__(128) uint8_t smem[];
  float *heads_smem = reinterpret_cast<float *>(smem + C::kSmemRing);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmemRing + C::kSmemHeads);
  int *prefix = reinterpret_cast<int *>(bars + kWarps * kStages);  // groups before sequence s
  int *part_seg = prefix + kMaxSeqs + 1;   // [2 * kWarps]: first and last part of each warp, -1: none
  int *part_flags = part_seg + 2 * kWarps;  // 1: has the segment's first group, 2: its last
  int *scan = part_flags + 2 * kWarps;      // [2 * kWarps]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t *wbar = bars + warp * kStages;
  uint8_t *ring = smem + warp * C::kRing;
  const int n = static_cast<int>(p.num_seqs);
  const int G = p.num_q_heads / p.num_kv_heads;
  const int H = p.num_kv_heads * tiles;  // segments of a sequence

  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(&wbar[s], 1);
    fence_mbar_init();
    part_seg[2 * warp] = part_seg[2 * warp + 1] = -1;
  }
  pdl_wait();

  // ---- groups of each sequence, their prefix sums and largest ----
  const int64_t cap = p.bt_stride * p.block_size;
  int c_max = 0;
  {
    constexpr int kPer = kMaxSeqs / (kWarps * 32);
    int c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = threadIdx.x * kPer + i;
      int ctx = s < n ? __ldg(p.context_lens + s) : 0;
      if (ctx > cap) {
        if (blockIdx.x == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
        ctx = static_cast<int>(cap);
      }
      c[i] = ctx > 0 ? (ctx - 1) / kMxGroup + 1 : 0;
      sum += c[i];
      c_max = max(c_max, c[i]);
    }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(kAll, incl, off);
      if (lane >= off) incl += v;
    }
    c_max = __reduce_max_sync(kAll, c_max);
    if (lane == 31) scan[warp] = incl, scan[kWarps + warp] = c_max;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      c_max = max(c_max, scan[kWarps + w]);
    }
    before += incl - sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = threadIdx.x * kPer + i;
      if (s < n) {
        prefix[s] = before;
        before += c[i];
        if (s == n - 1) prefix[n] = before;
      }
    }
    __syncthreads();
  }
  // sequences without a key: zeros
  for (int s = blockIdx.x; s < n; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    T *out = static_cast<T *>(p.out) + static_cast<int64_t>(s) * p.num_q_heads * D;
    for (int i = threadIdx.x * 8; i < p.num_q_heads * D; i += blockDim.x * 8)
      *reinterpret_cast<uint4 *>(out + i) = make_uint4(0u, 0u, 0u, 0u);
  }

  // ---- this warp's range of units (unit: one group of one segment) ----
  const uint32_t total = static_cast<uint32_t>(prefix[n]) * H;
  const uint32_t all_warps = gridDim.x * kWarps;
  uint32_t u0 = 0, u1 = 0;
  const uint32_t share = (total + all_warps - 1) / all_warps;
  if (static_cast<uint32_t>(n) * H <= gridDim.x &&
      static_cast<uint32_t>((c_max + kWarps - 1) / kWarps) <= share + kAlignedSlack) {
    if (blockIdx.x < static_cast<uint32_t>(n) * H) {  // one segment to a CTA
      const int s = blockIdx.x / H, c = prefix[s + 1] - prefix[s];
      const uint32_t base = static_cast<uint32_t>(prefix[s]) * H + (blockIdx.x - s * H) * c;
      u0 = base + static_cast<uint32_t>(c) * warp / kWarps;
      u1 = base + static_cast<uint32_t>(c) * (warp + 1) / kWarps;
    }
  } else {
    const uint64_t j = blockIdx.x * kWarps + warp;
    u0 = static_cast<uint32_t>(total * j / all_warps);
    u1 = static_cast<uint32_t>(total * (j + 1) / all_warps);
  }
  const int units = static_cast<int>(u1 - u0);

  // Unit u0 + i for lane-parallel use: its segment, group, and where its bytes are.
  struct Unit {
    int seq, ht, group, groups;
  };
  auto unit_of = [&](int i) -> Unit {
    const uint32_t u = u0 + i;
    const int per = static_cast<int>(u / H);
    int a = 0, b = n - 1;  // the last sequence whose prefix is not above `per`
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (prefix[mid] <= per)
        a = mid;
      else
        b = mid - 1;
    }
    Unit r;
    r.seq = a;
    r.groups = prefix[a + 1] - prefix[a];
    const int rest = static_cast<int>(u - static_cast<uint32_t>(prefix[a]) * H);
    r.ht = rest / r.groups;
    r.group = rest - r.ht * r.groups;
    return r;
  };
  const int per_page = p.block_size / kMxGroup;
  // A batch of 32 units, one per lane: the index of its group in the pools (-1: no
  // such page) and what `process` has to know: keys in the group (bits 0-4),
  // whether it is its segment's first (32) or last (64) group.
  auto load_batch = [&](int first, int &where, int &what) {
    where = -1, what = 0;
    const int i = first + lane;
    if (i >= units) return;
    const Unit r = unit_of(i);
    const int page = __ldg(p.block_tables + static_cast<int64_t>(r.seq) * p.bt_stride + r.group / per_page);
    int valid = kMxGroup;
    if (r.group == r.groups - 1) {
      const int ctx = static_cast<int>(min(static_cast<int64_t>(__ldg(p.context_lens + r.seq)), cap));
      valid = ctx - r.group * kMxGroup;
      what |= 64;
    }
    what |= valid | (r.group == 0 ? 32 : 0);
    if (page >= 0 && page < p.num_blocks)
      where = (page * p.num_kv_heads + r.ht / tiles) * per_page + r.group % per_page;
    else
      flag_status(p.status, MI_DEV_BAD_BLOCK);
  };
  int where_cur, what_cur, where_nxt, what_nxt;
  load_batch(0, where_cur, what_cur);
  load_batch(32, where_nxt, what_nxt);
  auto issue = [&](int now, int i) {  // unit i, while unit `now` is being worked on
    const int a = __shfl_sync(kAll, where_cur, i & 31), b = __shfl_sync(kAll, where_nxt, i & 31);
    const int where = (i >> 5) == (now >> 5) ? a : b;
    if (lane != 0) return;
    uint64_t *bar = &wbar[i % kStages];
    if (where < 0) {
      mbar_arrive(bar);
      return;
    }
    uint8_t *dst = ring + i % kStages * C::kStage;
    const int64_t off = static_cast<int64_t>(where) * C::kGroup;
    mbar_arrive_expect_tx(bar, C::kStage);
    bulk_g2s(dst, p.key_pages + off, C::kGroup, bar);
    bulk_g2s(dst + C::kGroup, p.value_pages + off, C::kGroup, bar);
  };
  int issued = 0;
  for (; issued < kStages && issued < units; ++issued) issue(0, issued);

  MxWarp<T, NB> st;
  st.lane = lane, st.g = lane >> 2, st.t = lane & 3;
  int seq = 0, ht = 0, heads = 0;
  bool has_first = false;
  auto start_segment = [&](int i) {
    const Unit r = unit_of(i);
    seq = r.seq, ht = r.ht;
    has_first = r.group == 0;
    const int kvh = ht / tiles, h0 = (ht - kvh * tiles) * kCols;
    heads = min(kCols, G - h0);
    st.reset();
    st.load_query(static_cast<const T *>(p.query) + (static_cast<int64_t>(seq) * p.num_q_heads + kvh * G + h0) * D,
                  heads, p.scale_log2);
  };
  auto end_segment = [&](bool has_last, bool final) {
    st.finish();
    if (has_first && has_last) {
      const int kvh = ht / tiles, h0 = (ht - kvh * tiles) * kCols;
      st.write_out(static_cast<T *>(p.out) + (static_cast<int64_t>(seq) * p.num_q_heads + kvh * G + h0) * D, heads);
      return;
    }
    const int slot = 2 * warp + (final ? 1 : 0);
    st.write_state(final ? reinterpret_cast<float *>(ring) : heads_smem + warp * C::kState, heads);
    if (lane == 0) {
      part_seg[slot] = seq * H + ht;
      part_flags[slot] = (has_first ? 1 : 0) | (has_last ? 2 : 0);
    }
  };

  bool timed_out = false;
#pragma unroll 1
  for (int i = 0; i < units; ++i) {
    const int what = __shfl_sync(kAll, what_cur, i & 31), where = __shfl_sync(kAll, where_cur, i & 31);
    if (i == 0 || (what & 32)) start_segment(i);
    if (!mbar_wait_bounded(&wbar[i % kStages], (i / kStages) & 1, p.status)) {
      timed_out = true;
      break;
    }
    if (where >= 0) {
      const uint32_t base = smem_addr(ring + i % kStages * C::kStage);
      st.process(base, base + C::kGroup, what & 31);
    }
    __syncwarp();  // every lane has read the stage
    const bool final = i == units - 1;
    if (issued < units) {
      issue(i, issued);
      ++issued;
    }
    if ((what & 64) || final) end_segment((what & 64) != 0, final);
    if ((i & 31) == 31) {  // the next unit starts batch (i + 1) / 32
      where_cur = where_nxt, what_cur = what_nxt;
      load_batch(i + 33, where_nxt, what_nxt);
    }
  }
  if (timed_out) {  // the copies in flight land before the ring is given up
    if (lane == 0)
      for (int k = max(0, issued - kStages); k < issued; ++k)
        if (!mbar_wait_bounded(&wbar[k % kStages], (k / kStages) & 1, p.status)) break;
    __syncwarp();
  }
  __syncthreads();

  // ---- join the parts: runs of one segment over neighbouring warps ----
  MxMeta meta = {-1, 0, -1, 0};
  float *ws = p.workspace + static_cast<int64_t>(blockIdx.x) * 2 * C::kState;
  auto part = [&](int k) -> const float * {
    return k & 1 ? reinterpret_cast<const float *>(smem + (k >> 1) * C::kRing) : heads_smem + (k >> 1) * C::kState;
  };
  for (int k = 0; k < 2 * kWarps;) {
    const int seg = part_seg[k];
    if (seg < 0) {
      ++k;
      continue;
    }
    int end = k, flags = 0;
    for (; end < 2 * kWarps && (part_seg[end] == seg || part_seg[end] < 0); ++end)
      if (part_seg[end] >= 0) flags |= part_flags[end];
    const int s = seg / H, h_t = seg - s * H, kvh = h_t / tiles, h0 = (h_t - kvh * tiles) * kCols;
    const int hs = min(kCols, G - h0);
    float *state = flags & 1 ? ws + C::kState : ws;  // began here / in an earlier CTA
    T *out = static_cast<T *>(p.out) + (static_cast<int64_t>(s) * p.num_q_heads + kvh * G + h0) * D;
    for (int e = threadIdx.x; e < hs * D; e += blockDim.x) {
      const int h = e / D;
      float M = -INFINITY, L = 0.f, A = 0.f;
      for (int w = k; w < end; ++w)
        if (part_seg[w] >= 0) M = fmaxf(M, part(w)[kCols * D + h]);
      for (int w = k; w < end; ++w) {
        if (part_seg[w] < 0) continue;
        const float *x = part(w);
        const float f = part_factor(x[kCols * D + h], x[kCols * D + kCols + h], M);
        L += f * x[kCols * D + kCols + h];
        A += f * x[e];
      }
      if (flags == 3) {
        out[e] = Elem<T>::from_float(L == 0.f ? 0.f : A / L);
      } else {
        state[e] = A;
        if (e - h * D == 0) state[kCols * D + h] = M, state[kCols * D + kCols + h] = L;
      }
    }
    if (flags != 3) {
      if (flags & 1)
        meta.tail = seg;
      else
        meta.head = seg, meta.head_ends = flags >> 1;
    }
    k = end;
  }
  if (threadIdx.x == 0 && p.workspace != nullptr)
    reinterpret_cast<MxMeta *>(p.workspace + static_cast<int64_t>(gridDim.x) * 2 * C::kState)[blockIdx.x] = meta;
  pdl_launch_dependents();
}

// Segments that cross CTAs: the CTA in which one begins joins it.
template <typename T, int NB>
__global__ void __launch_bounds__(512) mxfp4_decode_mma_join_kernel(const MxDecodeParams p, int tiles) {
  using C = MxCfg<NB>;
  constexpr int D = C::D;
  pdl_wait();
  const int ctas = gridDim.x;
  const MxMeta *meta = reinterpret_cast<const MxMeta *>(p.workspace + static_cast<int64_t>(ctas) * 2 * C::kState);
  const int first = blockIdx.x, seg = meta[first].tail;
  if (seg >= 0) {
    int end = first + 1;  // one past the last CTA that has a part
    while (end < ctas && meta[end].head == seg) {
      ++end;
      if (meta[end - 1].head_ends) break;
    }
    const int G = p.num_q_heads / p.num_kv_heads, H = p.num_kv_heads * tiles;
    const int s = seg / H, h_t = seg - s * H, kvh = h_t / tiles, h0 = (h_t - kvh * tiles) * kCols;
    const int hs = min(kCols, G - h0);
    T *out = static_cast<T *>(p.out) + (static_cast<int64_t>(s) * p.num_q_heads + kvh * G + h0) * D;
    auto part = [&](int c) { return p.workspace + (static_cast<int64_t>(c) * 2 + (c == first ? 1 : 0)) * C::kState; };
    for (int e = threadIdx.x; e < hs * D; e += blockDim.x) {
      const int h = e / D;
      float M = -INFINITY, L = 0.f, A = 0.f;
      for (int c = first; c < end; ++c) M = fmaxf(M, part(c)[kCols * D + h]);
      for (int c = first; c < end; ++c) {
        const float *x = part(c);
        const float f = part_factor(x[kCols * D + h], x[kCols * D + kCols + h], M);
        L += f * x[kCols * D + kCols + h];
        A += f * x[e];
      }
      out[e] = Elem<T>::from_float(L == 0.f ? 0.f : A / L);
    }
  }
  pdl_launch_dependents();
}

template <typename T, int NB>
cudaError_t launch_mma(const MxDecodeParams &p, int tiles, bool join, int ctas, cudaStream_t stream) {
  using C = MxCfg<NB>;
  auto kern = mxfp4_decode_mma_kernel<T, NB>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(kWarps * 32), C::kSmem, stream, p, tiles);
  if (e == cudaSuccess && join)
    e = launch_pdl(mxfp4_decode_mma_join_kernel<T, NB>, dim3(ctas), dim3(512), 0, stream, p, tiles);
  return e;
}

int mma_tiles(int num_q_heads, int num_kv_heads) { return (num_q_heads / num_kv_heads + kCols - 1) / kCols; }

// Whether some lengths that the table can hold need the second launch: not when
// every segment has a CTA and a full table is no more than the slack per warp.
bool mma_joins(int64_t num_seqs, int num_q_heads, int num_kv_heads, int64_t capacity, int sms) {
  const int64_t segments = num_seqs * num_kv_heads * mma_tiles(num_q_heads, num_kv_heads);
  return segments > sms || capacity > static_cast<int64_t>(kAlignedSlack) * kWarps * kMxGroup;
}

}  // namespace

// Shapes of this kernel: 32-bit unit and group counts, sequences in one launch's reach.
bool mxfp4_mma_supported(int dtype, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_blocks,
                         int block_size, int64_t capacity) {
  if (dtype != MI_DTYPE_BFLOAT16 && dtype != MI_DTYPE_FLOAT16) return false;
  if (head_dim != 64 && head_dim != 128) return false;
  const int64_t H = static_cast<int64_t>(num_kv_heads) * mma_tiles(num_q_heads, num_kv_heads);
  return num_blocks * num_kv_heads * (block_size / kMxGroup) < (int64_t{1} << 31) &&
         (capacity / kMxGroup + 1) * H < (int64_t{1} << 31);
}

size_t mxfp4_mma_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t capacity,
                           int sms) {
  if (!mma_joins(num_seqs, num_q_heads, num_kv_heads, capacity, sms)) return 0;
  return static_cast<size_t>(sms) * (2 * kCols * (head_dim + 2) * sizeof(float) + sizeof(MxMeta));
}

cudaError_t launch_mxfp4_mma(const MxDecodeParams &p, int dtype, cudaStream_t stream) {
  const int tiles = mma_tiles(p.num_q_heads, p.num_kv_heads), sms = sm_count_current();
  const int64_t capacity = p.bt_stride * p.block_size;
  const int64_t H = static_cast<int64_t>(p.num_kv_heads) * tiles;
  int64_t slice = ((int64_t{1} << 31) - 1) / ((capacity / kMxGroup + 1) * H);  // units stay in 32 bits
  if (slice > kMaxSeqs) slice = kMaxSeqs;
  for (int64_t s = 0; s < p.num_seqs; s += slice) {
    MxDecodeParams q = p;
    q.num_seqs = p.num_seqs - s < slice ? p.num_seqs - s : slice;
    const int64_t row = s * p.num_q_heads * p.head_dim * 2;
    q.query = static_cast<const char *>(p.query) + row;
    q.out = static_cast<char *>(p.out) + row;
    q.block_tables = p.block_tables + s * p.bt_stride;
    q.context_lens = p.context_lens + s;
    const bool join = mma_joins(p.num_seqs, p.num_q_heads, p.num_kv_heads, capacity, sms);
    cudaError_t e;
    if (dtype == MI_DTYPE_BFLOAT16)
      e = p.head_dim == 64 ? launch_mma<__nv_bfloat16, 2>(q, tiles, join, sms, stream)
                           : launch_mma<__nv_bfloat16, 4>(q, tiles, join, sms, stream);
    else
      e = p.head_dim == 64 ? launch_mma<__half, 2>(q, tiles, join, sms, stream)
                           : launch_mma<__half, 4>(q, tiles, join, sms, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mi
