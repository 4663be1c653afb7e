// Paged decode over the 8-bit cache (layout: fp8.cuh) on the warp-level tensor cores: one query token per sequence,
// out = softmax(scale * K q) V, any type, head_dim and GQA group.  Work, ring and joins: decode_segments.cuh.
//
// Decode moves a byte per cached element and does 2 flops per element and query head on it: HBM-bound as
// long as turning codes into MMA operands stays cheap.
//   - Two e4m3 bytes become an f16 pair in one instruction, and no scale meets an element: a group of 16
//     keys has one, so it multiplies 16 keys' scores (K) and goes into 16 keys' p (V).
//   - The pages hold the operands in the order of the lanes: a lane's 16 bytes of a part of 64 dims are, as they are,
//     its share of four m16n8k16 A fragments, K's rows (keys) with dims in an order that q follows, or V's transposed, two
//     neighbouring keys side by side.  So shared memory is read in whole 512-byte rows and no code moves between lanes.
//   - S^T = K Q^T (16 keys x 8 query heads), P^T through movmatrix, O^T += V^T P^T (16 dims x 8 query heads).  For fp32 the
//     8 columns are the upper and the lower f16 of 4 query heads, in S and in P, 22 bits together.
//   - V's scale: O is held in units of 2^(R - 127), R a running reference at or above the group's byte, and p goes in as
//     p * 2^(byte - R) * 2^12 in f16 (m lags the largest score by 3 binades at most, so below 2^15): a key
//     2^-19 of the largest keeps all its bits 7 binades below R.  A group further below is multiplied on its own and
//     added in fp32; a group above raises R.  R is the same for the whole warp.
//   - q is multiplied by a power of two that puts its largest element into [2^14, 2^15) and converted to f16
//     (exact for bf16 down to 2^-28 of that element); that power, K's scale and the softmax's scale become
//     one factor, put together from exponents so that it leaves fp32's range only where the scores do.
// Measured: 32 x 8192, 32 heads on 8 of 128, bf16: 99 us, 5.75 TB/s (88% of a copy), ALU 39%, issue slots 38%; 128 ragged up to 6000
// 147 us (166 with rings of 16-byte cp.async), 1 x 100001 44, 1 x 300 7.1 (10.8 as called; 14.7 with a join behind every call).
#include <type_traits>

#include "common.cuh"
#include "decode_segments.cuh"
#include "fp8.cuh"

namespace mi {

namespace {

constexpr float kLift = 12.f;  // p is held as 2^(x - m + kLift)
constexpr float kLag = 3.f;    // m may be this far behind: p <= 2^15
constexpr float kExact = 0x1p20f;  // m up to here is off by 2^-4 at most
constexpr int kNear = 7;       // binades below R that p takes in
constexpr int kFactorMax = 94; // largest exponent of a score's first factor: sums of products are below 2^32, and the
                               // scale's mantissa below 2

// Heads of a segment (CT column tiles of 8 columns: 8 query heads, fp32 4), and warps of a CTA: as many as shared memory
// holds with rings of two units.
constexpr int f8_heads(int columns, bool split) { return columns * (split ? 4 : 8); }
constexpr int f8_warps(int head_dim, int columns, bool split) {
  const int heads = f8_heads(columns, split);
  const int per_warp = 2 * 4 * f8_group_bytes(head_dim) + heads * (head_dim + 2) * 4 + 64 * 16 + 2 * 8 + 24 + 2 * heads * 12;
  const int fit = (227 * 1024 - (kMaxSeqs + 1) * 4 - 16) / per_warp;
  return fit > 16 ? 16 : fit;
}
constexpr int kF8Slack = 3;  // units per warp that keeping a segment in one CTA may cost: the second launch costs as much
// NB blocks of 32 dims.  q's fragments stay in registers.
template <int NB, int CT, bool SPLIT>
using F8Cfg = SegCfg<NB * 32, f8_warps(NB * 32, CT, SPLIT), 2, f8_heads(CT, SPLIT), f8_group_bytes(NB * 32), 0>;

__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(addr));
  return r;
}
template <int WORDS>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&w)[4]) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}
template <int WORDS>
__device__ __forceinline__ void sts(uint32_t addr, const uint32_t (&w)[4]) {
  if constexpr (WORDS == 4)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  else
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(w[0]), "r"(w[1]) : "memory");
}

// A warp's state on a segment, lane (g, t) = (lane / 4, lane % 4).
template <typename T, int NB, int CT>
struct F8Warp {
  using Elem_ = T;
  static constexpr int kSlack = kF8Slack;
  static constexpr bool kBulk = true;
  static constexpr bool kSplit = std::is_same<T, float>::value;
  using C = F8Cfg<NB, CT, kSplit>;
  static constexpr int D = C::D;
  static constexpr int kCols = kSplit ? 1 : 2;  // query heads of this lane in a tile: kCols * t and on
  static constexpr int kTileHeads = 4 * kCols;
  static constexpr int kCodes = kF8Group * D;   // bytes of a group's codes
  static constexpr int kFull = NB / 2;          // parts of 64 dims
  static constexpr int kOut = 2 * NB;           // 16-dim tiles of O: part p's are 4p to 4p + 3, a last part of 32 has two
  uint32_t q[CT][NB][4];  // this lane's B fragments of q
  float unit[CT][kCols];  // takes a sum of products to the log2 domain, but for K's scale: 2^power * mantissa
  int power[CT][kCols];
  int top_byte[CT][kCols];  // of K's scales that may multiply it
  float mantissa;         // of the softmax's scale
  float o[CT][kOut][4];   // columns 2t and 2t + 1, dims 2i and 2i + 1 of the lane's in the part, times 2^(R - 127)
  float m[CT][kCols], l[CT][kCols];  // l: this lane's keys only
  int ref;                // R
  int lane, g, t;

  __device__ __forceinline__ void setup(uint32_t) { lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3; }

  __device__ __forceinline__ void reset() {
    ref = 0;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
      for (int i = 0; i < kOut; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
#pragma unroll
      for (int u = 0; u < kCols; ++u) m[c][u] = -INFINITY, l[c][u] = 0.f;
    }
  }

  // First dim of this lane's 8 in block b of 32.
  __device__ __forceinline__ int dims_of(int b) const {
    return b / 2 < kFull ? b / 2 * 64 + t * 16 + (b & 1) * 8 : b * 32 + t * 8;
  }

  // q of the segment's query heads (heads of them exist): this lane's elements ...
  static constexpr int kRaw = 8 * static_cast<int>(sizeof(T)) / 16;
  using Raw = uint4[CT][NB][kRaw];
  __device__ __forceinline__ void fetch_query(const T *query, int heads, Raw &raw) const {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int h = c * kTileHeads + (kSplit ? g >> 1 : g);
#pragma unroll
      for (int i = 0; i < NB * kRaw; ++i) {
        uint4 &v = raw[c][i / kRaw][i % kRaw];
        v = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads) v = reinterpret_cast<const uint4 *>(query + h * D + dims_of(i / kRaw))[i % kRaw];
      }
    }
  }
  // ... as f16 fragments.
  __device__ __forceinline__ void set_query(const Raw &raw, float scale_log2) {
    const F8Scale scale = f8_softmax_scale(scale_log2);
    mantissa = scale.mantissa;
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
      if (top >= 0x7f800000u || top == 0 || scale.sign == 0.f) e = 0;  // not finite: as it is; nor do zeros need a power
      e = min(e, 126);
      const float f = exp2i(e) * scale.sign;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[b][i] *= f;
          if (kSplit && (g & 1)) x[b][i] -= __half2float(__float2half_rn(x[b][i]));  // what the other column leaves
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) q[c][b][i] = pack_f16(x[b][2 * i], x[b][2 * i + 1]);
      }
#pragma unroll
      for (int u = 0; u < kCols; ++u) {  // a lane of this query head: its column is 2t + u
        const int e2 = scale.exponent - __shfl_sync(kAll, e, 4 * (2 * t + u));
        power[c][u] = e2;
        const bool normal = e2 >= -126 && e2 <= kFactorMax;
        unit[c][u] = __uint_as_float(static_cast<uint32_t>((normal ? e2 : 0) + 127) << 23) * mantissa;
        top_byte[c][u] = normal ? kFactorMax + 127 - e2 : -1;
      }
    }
  }

  // S^T of part `part` (W words of codes a lane and row) of both groups.
  template <int W>
  __device__ __forceinline__ void score_part(uint32_t kbase, int part, float (&d)[2][CT][4]) const {
    uint32_t lo[2][4], hi[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t at = kbase + j * C::kGroup + part * 64 * kF8Group + lane * (4 * W);
      lds<W>(at, lo[j]);
      lds<W>(at + 128 * W, hi[j]);
    }
#pragma unroll
    for (int b = 0; b < W / 2; ++b) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t a[4];
          f8_to_f16(lo[j][2 * b + i], a[0], a[2]);
          f8_to_f16(hi[j][2 * b + i], a[1], a[3]);
#pragma unroll
          for (int c = 0; c < CT; ++c) mma_f16(d[j][c], a[0], a[1], a[2], a[3], q[c][2 * part + b][2 * i], q[c][2 * part + b][2 * i + 1]);
        }
    }
  }

  // Sums of products of a unit's 32 keys: x[j][c][r][u], key g + 8r of group j, query head kCols * t + u of tile c; and the
  // factors that make them scores in the log2 domain.
  __device__ __forceinline__ void scores(uint32_t kbase, float (&x)[2][CT][2][kCols], float (&factor)[2][CT][kCols]) const {
    float d[2][CT][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < CT; ++c) d[j][c][0] = d[j][c][1] = d[j][c][2] = d[j][c][3] = 0.f;
    const uint32_t byte[2] = {lds8(kbase + kCodes), lds8(kbase + C::kGroup + kCodes)};
#pragma unroll
    for (int p = 0; p < kFull; ++p) score_part<4>(kbase, p, d);
    if constexpr (NB % 2 != 0) score_part<2>(kbase, kFull, d);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
          x[j][c][0][u] = kSplit ? d[j][c][0] + d[j][c][1] : d[j][c][u];
          x[j][c][1][u] = kSplit ? d[j][c][2] + d[j][c][3] : d[j][c][2 + u];
          // further down every score is 0; not 0 itself, which a masked score would make a NaN
          factor[j][c][u] = fmaxf(f8_scale(byte[j]) * unit[c][u], 0x1p-126f);
          if (static_cast<int>(byte[j]) > top_byte[c][u]) {  // hardly ever
            const int e = byte[j] == 0 ? -126 : static_cast<int>(byte[j]) - 127 + power[c][u], near = max(-126, min(kFactorMax, e));
            factor[j][c][u] = __uint_as_float(static_cast<uint32_t>(near + 127) << 23) * mantissa;
            const float f = exp2i(max(0, e - kFactorMax));
            x[j][c][0][u] *= f, x[j][c][1][u] *= f;
          }
        }
  }

  // V's codes of keys from `valid` on become zeros, whatever they are: this lane's own, which no other reads.
  template <int W>
  __device__ __forceinline__ void clear_part(uint32_t at, int valid) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = 8 * h + 2 * t;
      const uint32_t keep = (key < valid ? 0x00ff00ffu : 0u) | (key + 1 < valid ? 0xff00ff00u : 0u);
      uint32_t w[4];
      lds<W>(at + h * 128 * W + lane * (4 * W), w);
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] &= keep;
      sts<W>(at + h * 128 * W + lane * (4 * W), w);
    }
  }
  __device__ __forceinline__ void clear_values(uint32_t vbase, int valid) const {
#pragma unroll
    for (int p = 0; p < kFull; ++p) clear_part<4>(vbase + p * 64 * kF8Group, valid);
    if constexpr (NB % 2 != 0) clear_part<2>(vbase + kFull * 64 * kF8Group, valid);
  }

  // O^T += V^T P^T of part `part` of a group.  FAR: the products are taken `back` times.
  template <int W, bool FAR>
  __device__ __forceinline__ void value_part(uint32_t vbase, int part, const uint32_t (&p)[CT][2], float back) {
    uint32_t h0[4], h1[4];
    const uint32_t at = vbase + part * 64 * kF8Group + lane * (4 * W);
    lds<W>(at, h0);
    lds<W>(at + 128 * W, h1);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t a[4];
      f8_to_f16(h0[i], a[0], a[1]);
      f8_to_f16(h1[i], a[2], a[3]);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if constexpr (FAR) {
          float r[4];
          mma_f16_zero(r, a[0], a[1], a[2], a[3], p[c][0], p[c][1]);
#pragma unroll
          for (int u = 0; u < 4; ++u) o[c][part * 4 + i][u] = fmaf(r[u], back, o[c][part * 4 + i][u]);
        } else {
          mma_f16(o[c][part * 4 + i], a[0], a[1], a[2], a[3], p[c][0], p[c][1]);
        }
      }
    }
  }
  template <bool FAR>
  __device__ __forceinline__ void values(uint32_t vbase, const uint32_t (&p)[CT][2], float back = 1.f) {
#pragma unroll
    for (int part = 0; part < kFull; ++part) value_part<4, FAR>(vbase, part, p, back);
    if constexpr (NB % 2 != 0) value_part<2, FAR>(vbase, kFull, p, back);
  }

  // One unit: K of its two groups at `base`, then V of both; `valid0` and `valid1` of their 16 keys exist; `special`:
  // that may be fewer than 16, or it is the `first` that the state meets.
  __device__ __forceinline__ void process(uint32_t base, bool special, int valid0, int valid1, bool first) {
    const uint32_t vbase = base + 2 * C::kGroup;
    float x[2][CT][2][kCols], factor[2][CT][kCols];
    scores(base, x, factor);
    int byte[2] = {static_cast<int>(lds8(vbase + kCodes)), static_cast<int>(lds8(vbase + C::kGroup + kCodes))};
    if (special) {  // uniform
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int valid = j ? valid1 : valid0;
        if (valid >= kF8Group) continue;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int u = 0; u < kCols; ++u) {
            if (g >= valid) x[j][c][0][u] = -INFINITY;
            if (g + 8 >= valid) x[j][c][1][u] = -INFINITY;
          }
        clear_values(vbase + j * C::kGroup, valid);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the copies that overwrite it
        if (valid <= 0) byte[j] = 0;
      }
      if (first) ref = max(byte[0], byte[1]) + 2;  // two binades of room
    }
    // m follows the largest score, up to kLag binades behind it (by the difference: m + kLag may round to m + 4 from 2^24 on)
    float top[CT][kCols];
    bool behind = false;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int u = 0; u < kCols; ++u) {
        top[c][u] = fmaxf(fmaxf(x[0][c][0][u], x[0][c][1][u]) * factor[0][c][u],
                          fmaxf(x[1][c][0][u], x[1][c][1][u]) * factor[1][c][u]);
        behind |= top[c][u] - m[c][u] > kLag;
      }
    if (__any_sync(kAll, behind)) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
          float mx = top[c][u];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, off));
          if (mx > m[c][u]) {  // the lanes of a query head agree
            const float f = m[c][u] == -INFINITY ? 0.f : fast_exp2(m[c][u] - mx);
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
              o[c][i][u] *= f, o[c][i][2 + u] *= f;
              if (kSplit) o[c][i][1] *= f, o[c][i][3] *= f;
            }
            l[c][u] *= f;
            m[c][u] = mx;
          }
        }
    }
    // V's scales: R not below them, and where they lie
    if (max(byte[0], byte[1]) > ref) {  // uniform, as all of this
      const int next = max(byte[0], byte[1]) + 2;
      const float f = exp2i(ref - next);
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < kOut * 4; ++i) o[c][i / 4][i % 4] *= f;
      ref = next;
    }
    float near[2];
    bool far[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      far[j] = byte[j] != 0 && ref - byte[j] > kNear;
      near[j] = byte[j] == 0 ? 0.f : far[j] ? 1.f : __uint_as_float(static_cast<uint32_t>(127 + byte[j] - ref) << 23);
    }
    uint32_t p[2][CT][2];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float lift[kCols];
      bool large = false;
#pragma unroll
      for (int u = 0; u < kCols; ++u) {
        lift[u] = kLift - m[c][u];
        large |= fabsf(m[c][u]) > kExact;
      }
      if (large) {  // m rounds away more than p may be off by: the products round as it did, and m goes at once
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i / 2][c][i % 2][u] = __fmul_rn(x[i / 2][c][i % 2][u], factor[i / 2][c][u]) - m[c][u];
          factor[0][c][u] = factor[1][c][u] = 1.f;
          lift[u] = kLift;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float w[2];
#pragma unroll
          for (int u = 0; u < kCols; ++u) {
            w[u] = fast_exp2(fmaf(x[j][c][r][u], factor[j][c][u], lift[u]));
            l[c][u] += w[u];
            w[u] *= near[j];
          }
          if constexpr (kSplit) w[1] = w[0] - __half2float(__float2half_rn(w[0]));
          // rows (keys) x columns, transposed: keys 2t and 2t + 1 of column g
          p[j][c][r] = movm(pack_f16(w[0], w[1]));
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (far[j])
        values<true>(vbase + j * C::kGroup, p[j], exp2i(byte[j] - ref));
      else
        values<false>(vbase + j * C::kGroup, p[j]);
    }
  }

  // Sum l over the keys of the lanes.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int u = 0; u < kCols; ++u)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[c][u] += __shfl_xor_sync(kAll, l[c][u], off);
  }

  // The mean of V over the keys seen, N of this lane's dims of a part from tile `tile` on: o is divided by l, which holds the
  // lift of p as o does, before the scale comes back, so that the result is in range where V is.
  template <int N>
  __device__ __forceinline__ void mean(int c, int u, int tile, float (&v)[8]) const {
    const float inv = l[c][u] == 0.f ? 0.f : __fdividef(1.f, l[c][u]), f = exp2i(ref - 127);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float *r = o[c][tile + i / 2] + 2 * (i & 1);
      v[i] = (kSplit ? r[0] + r[1] : r[u]) * inv * f;
    }
  }
  // store(row of the segment, dim, N, values) for each run of this lane's dims.
  template <typename F>
  __device__ __forceinline__ void each_run(int heads, F store) const {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int u = 0; u < kCols; ++u) {
        const int h = c * kTileHeads + kCols * t + u;
        if (h >= heads) continue;
        float v[8];
#pragma unroll
        for (int p = 0; p < kFull; ++p) {
          mean<8>(c, u, 4 * p, v);
          store(h, p * 64 + g * 8, std::integral_constant<int, 8>{}, v);
        }
        if constexpr (NB % 2 != 0) {
          mean<4>(c, u, 4 * kFull, v);
          store(h, kFull * 64 + g * 4, std::integral_constant<int, 4>{}, v);
        }
      }
  }

  __device__ __forceinline__ void write_out(T *out, int heads) const {
    each_run(heads, [&](int h, int dim, auto n, const float (&v)[8]) {
      constexpr int kVec = kSplit ? 4 : decltype(n)::value;
#pragma unroll
      for (int i = 0; i < decltype(n)::value; i += kVec) {
        using V = typename std::conditional<kVec * sizeof(T) == 16, uint4, uint2>::type;
        V w;
        T *e = reinterpret_cast<T *>(&w);
#pragma unroll
        for (int k = 0; k < kVec; ++k) e[k] = Elem<T>::from_float(v[i + k]);
        *reinterpret_cast<V *>(out + h * D + dim + i) = w;
      }
    });
  }

  __device__ __forceinline__ void write_state(float *st, int heads) const {
    each_run(heads, [&](int h, int dim, auto n, const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < decltype(n)::value; i += 4)
        *reinterpret_cast<float4 *>(st + h * D + dim + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    });
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int u = 0; u < kCols; ++u) {
        const int h = c * kTileHeads + kCols * t + u;
        if (h >= heads || g != 0) continue;
        st[C::kHeads * D + h] = m[c][u];
        st[C::kHeads * D + C::kHeads + h] = l[c][u];
      }
  }
};

template <typename T, int NB, int CT>
__global__ void __launch_bounds__(F8Warp<T, NB, CT>::C::kWarps * 32, 1)
    fp8_decode_kernel(const CodedDecodeParams p, const SegPlan plan) {
  decode_segments<F8Warp<T, NB, CT>>(p, plan);
}

template <typename T, int NB, int CT>
__global__ void __launch_bounds__(kJoinLanes * kJoinWays)
    fp8_decode_join_kernel(const CodedDecodeParams p, const SegPlan plan) {
  join_segments<F8Warp<T, NB, CT>>(p, plan);
}

template <typename T, int NB, int CT>
cudaError_t launch_f8(const CodedDecodeParams &p, int tiles, bool join, int ctas, cudaStream_t stream) {
  return launch_segments<F8Warp<T, NB, CT>>(fp8_decode_kernel<T, NB, CT>, fp8_decode_join_kernel<T, NB, CT>, p, tiles,
                                            join, ctas, stream);
}

// Column tiles of a segment (two rings' worth of sums do not fit past D = 128), and segments of a kv head.
int f8_columns(int group, int head_dim, bool split) { return group <= f8_heads(1, split) || head_dim > 128 ? 1 : 2; }
int f8_tiles(int group, int head_dim, bool split) {
  const int heads = f8_heads(f8_columns(group, head_dim, split), split);
  return (group + heads - 1) / heads;
}

bool f8_joins(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, bool split, int64_t capacity, int sms) {
  const int group = num_q_heads / num_kv_heads;
  return segments_join(num_seqs * num_kv_heads * f8_tiles(group, head_dim, split), capacity,
                       kF8Slack * f8_warps(head_dim, f8_columns(group, head_dim, split), split), sms);
}

template <typename T>
cudaError_t launch_f8_t(const CodedDecodeParams &p, int tiles, int columns, bool join, int ctas, cudaStream_t stream) {
  switch (p.head_dim / 32 * 2 + columns) {
    case 3: return launch_f8<T, 1, 1>(p, tiles, join, ctas, stream);
    case 4: return launch_f8<T, 1, 2>(p, tiles, join, ctas, stream);
    case 5: return launch_f8<T, 2, 1>(p, tiles, join, ctas, stream);
    case 6: return launch_f8<T, 2, 2>(p, tiles, join, ctas, stream);
    case 7: return launch_f8<T, 3, 1>(p, tiles, join, ctas, stream);
    case 8: return launch_f8<T, 3, 2>(p, tiles, join, ctas, stream);
    case 9: return launch_f8<T, 4, 1>(p, tiles, join, ctas, stream);
    case 10: return launch_f8<T, 4, 2>(p, tiles, join, ctas, stream);
    case 11: return launch_f8<T, 5, 1>(p, tiles, join, ctas, stream);
    case 13: return launch_f8<T, 6, 1>(p, tiles, join, ctas, stream);
    case 15: return launch_f8<T, 7, 1>(p, tiles, join, ctas, stream);
    case 17: return launch_f8<T, 8, 1>(p, tiles, join, ctas, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

bool fp8_decode_supported(int num_q_heads, int num_kv_heads, int head_dim, int dtype, int64_t num_blocks, int block_size,
                          int64_t capacity) {
  const int tiles = f8_tiles(num_q_heads / num_kv_heads, head_dim, dtype == MI_DTYPE_FLOAT32);
  return segments_supported(static_cast<int64_t>(num_kv_heads) * tiles, num_kv_heads, num_blocks, block_size, capacity);
}

size_t fp8_decode_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                            int64_t capacity, int sms) {
  const bool split = dtype == MI_DTYPE_FLOAT32;
  sms = segment_ctas(sms);
  if (!f8_joins(num_seqs, num_q_heads, num_kv_heads, head_dim, split, capacity, sms)) return 0;
  return segment_workspace(f8_heads(f8_columns(num_q_heads / num_kv_heads, head_dim, split), split), head_dim, sms);
}

cudaError_t launch_fp8_decode(const CodedDecodeParams &p, int dtype, cudaStream_t stream) {
  const int group = p.num_q_heads / p.num_kv_heads;
  const bool split = dtype == MI_DTYPE_FLOAT32;
  const int tiles = f8_tiles(group, p.head_dim, split), columns = f8_columns(group, p.head_dim, split);
  const int sms = segment_ctas(sm_count_current());
  const bool join =
      f8_joins(p.num_seqs, p.num_q_heads, p.num_kv_heads, p.head_dim, split, p.bt_stride * p.block_size, sms);
  return launch_segment_slices(p, tiles, dtype, [&](const CodedDecodeParams &q) {
    return dtype == MI_DTYPE_BFLOAT16 ? launch_f8_t<__nv_bfloat16>(q, tiles, columns, join, sms, stream)
           : dtype == MI_DTYPE_FLOAT16  ? launch_f8_t<__half>(q, tiles, columns, join, sms, stream)
                                        : launch_f8_t<float>(q, tiles, columns, join, sms, stream);
  });
}

}  // namespace mi
