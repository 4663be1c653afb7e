// Decode over quantised pages: the work list, the ring of copies and the joins that the formats share.
//
// One query token per sequence, out = softmax(scale * K q) V.  A page holds groups of 16 tokens of one kv head, K and V in
// C::kGroup contiguous bytes each; what they are is the business of W, a warp's state on a segment
// (a sequence, kv head and up to C::kHeads of its query heads):
//   W::C                      SegCfg of the format and shape
//   W::Elem_                  type of query and out
//   W::kSlack                 units per warp that keeping a segment in one CTA may cost
//   W::kBulk                  whether a lane fills the ring by bulk copies, or all by 16-byte ones
//   setup(shared address of C::kQuery bytes), fetch_query(), set_query(), reset()
//   process(base, special, valid0, valid1, first): one unit of 32 keys, K of its two groups at `base`, then V of both
//   finish(), write_out(), write_state(): the mean of V over the keys seen, and m and l
//
// Work: the units of 32 keys of all segments, in that order, are one list that is cut into equal ranges, one per
// warp (one CTA to an SM), so ragged batches and single long
// sequences load every SM alike.  A warp streams its range through a ring of its own, a few units
// deep, that runs across segment borders.  Segments that lie within one
// warp's range are written at once; the parts of others are joined in shared
// memory, and those that cross CTAs by a second launch, whose order is fixed.
// When every segment fits a CTA at hardly more work per warp, each CTA takes one
// segment and the second launch has nothing to do.
//
// Segments' results are means of V, divided by l before V's scale comes back, and are joined as means: nothing in
// between is larger than V itself.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "params.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kSegGroup = 16;           // tokens of a group
constexpr int kUnit = 2 * kSegGroup;    // keys of a unit of work
constexpr int kMaxSeqs = 2048;          // sequences of one launch (prefix sums in shared memory)

// Shared memory of a CTA of WARPS warps, each with a ring of STAGES units of GROUP-byte groups and QUERY bytes for q.
template <int D_, int WARPS, int STAGES, int HEADS, int GROUP, int QUERY>
struct SegCfg {
  static constexpr int D = D_;
  static constexpr int kWarps = WARPS;
  static constexpr int kStages = STAGES;
  static constexpr int kHeads = HEADS;            // query heads of a segment
  static constexpr int kGroup = GROUP;            // bytes of one group of one operand
  static constexpr int kStage = 4 * kGroup;       // K of two groups, V of two groups
  static constexpr int kRing = kStages * kStage;  // per warp
  static constexpr int kState = kHeads * (D + 2); // floats: mean of V [heads][D], m [heads], l [heads]
  static constexpr int kSmemRing = kWarps * kRing;
  static constexpr int kSmemHeads = kWarps * kState * 4;  // parts that end before their warp's range does
  static constexpr int kSmemUnits = kWarps * 64 * 16;     // two batches of 32 units per warp
  static constexpr int kQuery = QUERY;                    // q's fragments, per warp
  static constexpr int kSmemQuery = kWarps * kQuery;
  static constexpr int kSmemBars = kWarps * kStages * 8;  // bulk copies: a barrier to a stage
  static constexpr int kSmemPrefix = (kMaxSeqs + 1) * 4;
  static constexpr int kSmemMisc = 6 * kWarps * 4 + 2 * kWarps * kHeads * 12 + 16;
  static constexpr int kSmem = kSmemRing + kSmemHeads + kSmemUnits + kSmemQuery + kSmemBars + kSmemPrefix +
                               kSmemMisc;
  static_assert(kState * 4 <= kRing, "a warp's last part goes into its own ring");
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// Launch constants: tiles of a kv head (segments), and divisions by what the host knows.
struct SegPlan {
  int tiles;
  FastDiv by_segments;  // segments of a sequence: num_kv_heads * tiles
  FastDiv by_tiles;
  FastDiv by_page;      // groups of a page
  FastDiv by_ctas;
};

// Beside its states (a part whose segment began in an earlier CTA, then one whose
// segment goes on in the next) a CTA leaves in the workspace the segment that goes
// on (-1: none) and how many CTAs hold parts of it.
struct SegMeta {
  int32_t segment, parts;
};

// Where a CTA's join puts what its parts of a segment hold together, by their flags (1: the segment's first unit, 2: its last):
// into the result, or into one of the CTA's two states, which a call has only where a second launch was planned.  Without them
// every segment is whole, unless a wait gave up and its part is missing (the status says so): then there is nowhere to write.
enum class SegDest { kOut, kEarlier, kGoesOn, kNowhere };
__host__ __device__ constexpr SegDest segment_dest(int flags, bool states) {
  return flags == 3 ? SegDest::kOut : !states ? SegDest::kNowhere : (flags & 1) != 0 ? SegDest::kGoesOn : SegDest::kEarlier;
}
static_assert(segment_dest(3, false) == SegDest::kOut && segment_dest(3, true) == SegDest::kOut);
static_assert(segment_dest(0, false) == SegDest::kNowhere && segment_dest(1, false) == SegDest::kNowhere &&
              segment_dest(2, false) == SegDest::kNowhere);
static_assert(segment_dest(0, true) == SegDest::kEarlier && segment_dest(2, true) == SegDest::kEarlier &&
              segment_dest(1, true) == SegDest::kGoesOn);

__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 2^e for any e, through two factors where one has no normal exponent.
__device__ __forceinline__ float exp2i(int e) {
  const int a = max(-126, min(127, e)), b = max(-126, min(127, e - a));
  return __uint_as_float(static_cast<uint32_t>(a + 127) << 23) * __uint_as_float(static_cast<uint32_t>(b + 127) << 23);
}

// exp2(m - M) of a part: 0 for one without a key, 1 where both are -inf or NaN (l carries the NaN).
__device__ __forceinline__ float part_factor(float m, float l, float M) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return fast_exp2(m - M);
}
template <class W>
__device__ __forceinline__ void decode_segments(const CodedDecodeParams &p, const SegPlan &plan) {
  using C = typename W::C;
  using T = typename W::Elem_;
  constexpr int D = C::D, kWarps = C::kWarps, kStages = C::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  float *heads_smem = reinterpret_cast<float *>(smem + C::kSmemRing);
  int4 *unit_table = reinterpret_cast<int4 *>(smem + C::kSmemRing + C::kSmemHeads);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmemRing + C::kSmemHeads + C::kSmemUnits + C::kSmemQuery) +
                   (threadIdx.x >> 5) * C::kStages;
  int *prefix =
      reinterpret_cast<int *>(smem + C::kSmemRing + C::kSmemHeads + C::kSmemUnits + C::kSmemQuery + C::kSmemBars);  // units of a segment before sequence s
  int *part_seg = prefix + kMaxSeqs + 1;   // [2 * kWarps]: first and last part of each warp, -1: none
  int *part_flags = part_seg + 2 * kWarps;  // 1: has the segment's first group, 2: its last
  int *scan = part_flags + 2 * kWarps;      // [2 * kWarps]
  int *part_at = scan;                      // [2 * kWarps] after the scan: offsets of the parts, in floats
  float *factor = reinterpret_cast<float *>(scan + 2 * kWarps);  // [2 * kWarps][heads]
  float2 *run_ml = reinterpret_cast<float2 *>(                   // [2 * kWarps][heads]
      (reinterpret_cast<uintptr_t>(factor + 2 * kWarps * C::kHeads) + 15) & ~static_cast<uintptr_t>(15));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t *ring = smem + warp * C::kRing;
  const int n = static_cast<int>(p.num_seqs);
  const int G = p.num_q_heads / p.num_kv_heads;
  const int tiles = plan.tiles, H = p.num_kv_heads * tiles;  // segments of a sequence

  if constexpr (W::kBulk) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) mbar_init(bars + i, 1);
      fence_mbar_init();
    }
    __syncwarp();
  }
  pdl_wait();

  // ---- units of each sequence, their prefix sums and largest ----
  const int64_t cap = p.bt_stride * p.block_size;
  int c_max = 0;
  auto units_of = [&](int s) {
    int ctx = s < n ? __ldg(p.context_lens + s) : 0;
    if (ctx > cap) {
      if (blockIdx.x == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
      ctx = static_cast<int>(cap);
    }
    return ctx > 0 ? (ctx - 1) / kUnit + 1 : 0;
  };
  if (lane == 0) part_seg[2 * warp] = part_seg[2 * warp + 1] = -1;
  if (n <= 32) {  // every warp for itself
    const int c = units_of(lane);
    int incl = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(kAll, incl, off);
      if (lane >= off) incl += v;
    }
    c_max = __reduce_max_sync(kAll, c);
    if (warp == 0) {
      if (lane == 0) prefix[0] = 0;
      if (lane < n) prefix[lane + 1] = incl;
    }
  } else {
    constexpr int kPer = (kMaxSeqs + kWarps * 32 - 1) / (kWarps * 32);
    int c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      c[i] = units_of(threadIdx.x * kPer + i);
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
  }
  __syncthreads();
  // sequences without a key: zeros
  for (int s = blockIdx.x; s < n; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    T *out = static_cast<T *>(p.out) + static_cast<int64_t>(s) * p.num_q_heads * D;
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    for (int i = threadIdx.x * kVec; i < p.num_q_heads * D; i += blockDim.x * kVec)
      *reinterpret_cast<uint4 *>(out + i) = make_uint4(0u, 0u, 0u, 0u);
  }

  // ---- this CTA's range of units (a unit: 32 keys of one segment), split among its warps ----
  const uint32_t total = static_cast<uint32_t>(prefix[n]) * H;
  const uint32_t share = plan.by_ctas.div(total), over = total - share * gridDim.x;  // `over` CTAs take one more
  uint32_t u0, cta_units;
  if (static_cast<uint32_t>(n) * H <= gridDim.x &&
      static_cast<uint32_t>(c_max) <= share + (over != 0) + W::kSlack * kWarps) {
    const int s = static_cast<int>(plan.by_segments.div(blockIdx.x));  // one segment to a CTA
    cta_units = s < n ? prefix[s + 1] - prefix[s] : 0;
    u0 = s < n ? static_cast<uint32_t>(prefix[s]) * H + (blockIdx.x - s * H) * cta_units : 0;
  } else {
    cta_units = share + (blockIdx.x < over);
    u0 = share * blockIdx.x + min(blockIdx.x, over);
  }
  const int units = static_cast<int>(cta_units * (warp + 1) / kWarps - cta_units * warp / kWarps);
  u0 += cta_units * warp / kWarps;

  // Batches of 32 units, one per lane, in shared memory: x, y, the indices of the unit's two groups in
  // the pools (0 where there is none: every unit brings two); z, its keys (bits 0-5) and flags; w, its segment.
  constexpr int kStarts = 64;   // the warp's first unit of its segment
  constexpr int kEnds = 128;    // its last
  constexpr int kFirst = 256;   // the segment's first unit
  constexpr int kLast = 512;    // the segment's last
  constexpr int kNoPage = 1024; // its first group's page is none: flagged, left out (the second's is as if past the context)
  const int per_page = p.block_size / kSegGroup;
  int4 *table = unit_table + warp * 64;
  struct Unit {
    int seq, ht, unit, count;
  };
  auto unit_of = [&](int i) {
    const uint32_t u = u0 + i;
    const int per = static_cast<int>(plan.by_segments.div(u));
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
    r.count = prefix[a + 1] - prefix[a];
    const int rest = static_cast<int>(u - static_cast<uint32_t>(prefix[a]) * H);
    r.ht = static_cast<int>(__fdividef(static_cast<float>(rest), static_cast<float>(r.count)));  // off by one at most
    if (r.ht * r.count > rest) --r.ht;
    if (rest - r.ht * r.count >= r.count) ++r.ht;
    r.unit = rest - r.ht * r.count;
    return r;
  };
  auto load_batch = [&](int i, const Unit &r) {
    if (i < units) {
      int valid = kUnit, flags = 0;
      if (r.unit == 0) flags |= kStarts | kFirst;
      if (i == 0) flags |= kStarts;
      if (i == units - 1) flags |= kEnds;
      if (r.unit == r.count - 1) {
        const int ctx = static_cast<int>(min(static_cast<int64_t>(__ldg(p.context_lens + r.seq)), cap));
        valid = ctx - r.unit * kUnit;
        flags |= kEnds | kLast;
      }
      const int32_t *row = p.block_tables + static_cast<int64_t>(r.seq) * p.bt_stride;
      const int kvh = static_cast<int>(plan.by_tiles.div(r.ht));
      int where[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j * kSegGroup >= valid) break;
        const int group = 2 * r.unit + j, col = static_cast<int>(plan.by_page.div(group));
        const int page = __ldg(row + col);
        if (page >= 0 && page < p.num_blocks) {
          where[j] = (page * p.num_kv_heads + kvh) * per_page + group - col * per_page;
        } else {
          flag_status(p.status, MI_DEV_BAD_BLOCK);
          if (j == 0)
            flags |= kNoPage;
          else
            valid = kSegGroup;
        }
      }
      table[i & 63] = make_int4(where[0], where[1], valid | flags, r.seq * H + r.ht);
    }
    __syncwarp();
  };
  // Copies of unit i to stage `at`, K and V of its two groups: 16 bytes a lane, whole rows of 32 lanes,
  // then what is left of the four runs, in one where a row holds it.
  constexpr int kVecs = C::kGroup / 16, kFull = kVecs / 32, kLeft = kVecs % 32;
  const uint32_t my_place = smem_addr(ring) + lane * 16;
  const uint8_t *my_keys = p.key_pages + lane * 16, *my_values = p.value_pages + lane * 16;
  const int left_run = lane / kLeft, left_at = (kFull * 32 + lane % kLeft) * 16;
  const uint8_t *my_left = (left_run & 2 ? p.value_pages : p.key_pages) + left_at;
  const uint32_t my_left_place = smem_addr(ring) + left_run * C::kGroup + left_at;
  auto copy16 = [](uint32_t to, const uint8_t *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  };
  auto issue = [&](int i, int at) {
    const int2 where = *reinterpret_cast<const int2 *>(table + (i & 63));
    if constexpr (W::kBulk) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bars + at, C::kStage);
#pragma unroll
        for (int run = 0; run < 4; ++run)
          bulk_g2s(ring + at * C::kStage + run * C::kGroup,
                   (run & 2 ? p.value_pages : p.key_pages) + static_cast<int64_t>(run & 1 ? where.y : where.x) * C::kGroup,
                   C::kGroup, bars + at);
      }
      return;
    }
    const uint32_t to = my_place + at * C::kStage;
#pragma unroll
    for (int run = 0; run < 4; ++run) {
      const uint8_t *from = (run & 2 ? my_values : my_keys) + static_cast<int64_t>(run & 1 ? where.y : where.x) * C::kGroup;
#pragma unroll
      for (int v = 0; v < kFull; ++v) copy16(to + run * C::kGroup + v * 512, from + v * 512);
      if (kLeft > 8 && lane < kLeft) copy16(to + run * C::kGroup + kFull * 512, from + kFull * 512);
    }
    if (kLeft <= 8 && lane < 4 * kLeft)
      copy16(my_left_place + at * C::kStage,
             my_left + static_cast<int64_t>(left_run & 1 ? where.y : where.x) * C::kGroup);
  };
  auto commit = [] {
    if constexpr (!W::kBulk) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Whether unit i has come to stage `at` (else the status says so), the same for every lane: one whose wait gave up takes the
  // others with it.
  auto arrived = [&](int i, int at) {
    if constexpr (W::kBulk) {
      return __all_sync(kAll, mbar_wait_bounded(bars + at, i / kStages & 1, p.status)) != 0;
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");  // this lane's copies
      __syncwarp();                                                         // every lane's
      return true;
    }
  };

  W st;
  st.setup(smem_addr(smem + C::kSmemRing + C::kSmemHeads + C::kSmemUnits + warp * C::kQuery));
  int segment = 0, heads = 0;
  int64_t row = 0;  // the segment's first query head, as a row of q and out
  bool has_first = false;
  auto place = [&](int seg) {
    segment = seg;
    const int seq = static_cast<int>(plan.by_segments.div(seg)), ht = seg - seq * H;
    const int kvh = static_cast<int>(plan.by_tiles.div(ht)), h0 = (ht - kvh * tiles) * C::kHeads;
    heads = min(C::kHeads, G - h0);
    row = static_cast<int64_t>(seq) * p.num_q_heads + kvh * G + h0;
  };
  auto end_segment = [&](bool has_last, bool final) {
    st.finish();
    if (has_first && has_last) {
      st.write_out(static_cast<T *>(p.out) + row * D, heads);
      return;
    }
    const int slot = 2 * warp + (final ? 1 : 0);
    st.write_state(final ? reinterpret_cast<float *>(ring) : heads_smem + warp * C::kState, heads);
    if (lane == 0) {
      part_seg[slot] = segment;
      part_flags[slot] = (has_first ? 1 : 0) | (has_last ? 2 : 0);
    }
  };

  // The first segment's q is asked for before the ring's copies, which would keep it waiting.
  typename W::Raw raw;
  if (units > 0) {
    const Unit r = unit_of(min(lane, units - 1));
    place(__shfl_sync(kAll, r.seq * H + r.ht, 0));
    st.fetch_query(static_cast<const T *>(p.query) + row * D, heads, raw);
    load_batch(lane, r);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      if (i < units) issue(i, i);
      commit();
    }
    st.set_query(raw, p.scale_log2);
  }

  bool fresh = true;
  int stage = 0;
#pragma unroll 1
  for (int i = 0; i < units; ++i) {
    if ((i & 31) == 0 && i + 32 < units)  // into the half that units i - 32 to i - 1 have left
      load_batch(i + 32 + lane, unit_of(min(i + 32 + lane, units - 1)));
    const int4 unit = table[i & 63];
    const int what = unit.z;
    if (what & kStarts) {
      if (i > 0) {
        place(unit.w);
        st.fetch_query(static_cast<const T *>(p.query) + row * D, heads, raw);
        st.set_query(raw, p.scale_log2);
      }
      has_first = (what & kFirst) != 0;
      st.reset();
      fresh = true;
    }
    if (!arrived(i, stage)) {
      for (int k = i + 1; k < min(units, i + kStages); ++k) arrived(k, k % kStages);  // nothing is on its way at the end
      break;
    }
    const bool special = what != kUnit || fresh;
    const int valid = what & 63, valid0 = what & kNoPage ? 0 : min(valid, kSegGroup), valid1 = valid - kSegGroup;
    if (valid0 > 0 || valid1 > 0) {
      st.process(smem_addr(ring) + stage * C::kStage, special, valid0, valid1, fresh);
      fresh = false;
    }
    __syncwarp();  // every lane has read the stage
    if (i + kStages < units) issue(i + kStages, stage);
    commit();
    if (what & kEnds) end_segment((what & kLast) != 0, i == units - 1);
    if (++stage == kStages) stage = 0;
  }
  __syncthreads();

  // ---- join the parts: runs of one segment over neighbouring warps ----
  // Every warp sees the list of parts, one per lane; in shared memory they are without gaps.
  static_assert(2 * kWarps <= 32, "one lane per part");
  const int my_seg = lane < 2 * kWarps ? part_seg[lane] : -1;
  const unsigned present = __ballot_sync(kAll, my_seg >= 0);
  const unsigned below = present & ((1u << lane) - 1u);
  const int rank = __popc(below);
  const int prev_seg = __shfl_sync(kAll, my_seg, below ? 31 - __clz(below) : lane);
  const unsigned starts = __ballot_sync(kAll, my_seg >= 0 && (below == 0 || prev_seg != my_seg));
  const int my_flags = my_seg >= 0 ? part_flags[lane] : 0;
  const float *my_part = lane & 1 ? reinterpret_cast<const float *>(smem + (lane >> 1) * C::kRing)
                                  : heads_smem + (lane >> 1) * C::kState;
  if (warp == 0 && my_seg >= 0) part_at[rank] = static_cast<int>(my_part - reinterpret_cast<const float *>(smem));
  // their factors and sums: warp h takes query head h
  for (int h = warp; h < C::kHeads; h += kWarps) {
    float m = -INFINITY, l = 0.f;
    if (my_seg >= 0) m = my_part[C::kHeads * D + h], l = my_part[C::kHeads * D + C::kHeads + h];
    for (unsigned left = starts; left; left &= left - 1) {
      const int k = __ffs(left) - 1;
      const unsigned later = left & (left - 1);
      const bool mine = my_seg >= 0 && lane >= k && (later == 0 || lane < __ffs(later) - 1);
      float M = mine ? m : -INFINITY;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, off));
      const float f = mine ? part_factor(m, l, M) : 0.f;
      float L = mine ? f * l : 0.f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(kAll, L, off);
      if (mine) factor[rank * C::kHeads + h] = L == 0.f ? 0.f : __fdividef(f * l, L);  // its share of the mean
      if (lane == k) run_ml[rank * C::kHeads + h] = make_float2(M, L);
    }
  }
  __syncthreads();
  float *ws = p.workspace + static_cast<int64_t>(blockIdx.x) * 2 * C::kState;
  SegMeta meta = {-1, 0};
  bool has_head = false;
  for (unsigned left = starts; left; left &= left - 1) {
    const int k = __ffs(left) - 1;
    const unsigned later = left & (left - 1);
    const unsigned in_run = present & ~((1u << k) - 1u) & (later ? (1u << (__ffs(later) - 1)) - 1u : kAll);
    const int j0 = __popc(present & ((1u << k) - 1u)), j1 = j0 + __popc(in_run);
    const int flags = __reduce_or_sync(kAll, in_run >> lane & 1u ? my_flags : 0);
    place(__shfl_sync(kAll, my_seg, k));
    if (flags == 1) {  // goes on in later CTAs, up to the one that holds its last unit
      const int s = static_cast<int>(plan.by_segments.div(segment));
      const uint32_t last = static_cast<uint32_t>(prefix[s]) * H +
                            static_cast<uint32_t>(segment - s * H + 1) * (prefix[s + 1] - prefix[s]) - 1;
      const uint32_t edge = over * (share + 1);  // units of the CTAs that take one more
      const uint32_t cta = last < edge ? last / (share + 1) : over + (last - edge) / share;
      meta.segment = segment;
      meta.parts = static_cast<int>(cta - blockIdx.x) + 1;
    }
    const SegDest dest = segment_dest(flags, p.workspace != nullptr);
    if (dest == SegDest::kNowhere) continue;
    has_head |= dest == SegDest::kEarlier;
    float *state = dest == SegDest::kGoesOn ? ws + C::kState : ws;
    T *out = static_cast<T *>(p.out) + row * D;
    for (int e = threadIdx.x; e < heads * D; e += blockDim.x) {
      const int h = e / D;
      float A = 0.f;
#pragma unroll 4
      for (int j = j0; j < j1; ++j)
        A = fmaf(factor[j * C::kHeads + h], reinterpret_cast<const float *>(smem)[part_at[j] + e], A);
      if (dest == SegDest::kOut) {
        out[e] = Elem<T>::from_float(A);
      } else {
        state[e] = A;
        if (e - h * D == 0) {
          const float2 ml = run_ml[j0 * C::kHeads + h];
          state[C::kHeads * D + h] = ml.x, state[C::kHeads * D + C::kHeads + h] = ml.y;
        }
      }
    }
  }
  if (p.workspace != nullptr) {
    if (threadIdx.x == 0)
      reinterpret_cast<SegMeta *>(p.workspace + static_cast<int64_t>(gridDim.x) * 2 * C::kState)[blockIdx.x] = meta;
    if (!has_head && threadIdx.x < C::kHeads) {  // no part to give: one without keys
      ws[C::kHeads * D + threadIdx.x] = -INFINITY;
      ws[C::kHeads * D + C::kHeads + threadIdx.x] = 0.f;
    }
  }
  pdl_launch_dependents();
}


// Segments that cross CTAs: block c joins the one that goes on from CTA c.  A warp takes a query head's m and l,
// a lane to a part, and turns them into the parts' shares of the mean; then a thread takes 4 elements, the quarters of the
// block every fourth part.  The first parts are read while the block is still finding out whether they are
// any.  (Joining in the first launch, by the CTA that arrives last, took longer: its fences and the atomic
// cost 5 us at 1 x 131072, this launch 4.)
constexpr int kJoinWays = 4;
constexpr int kJoinLanes = 128;
constexpr int kMaxCtas = 192;  // of the first launch
template <class W>
__device__ __forceinline__ void join_segments(const CodedDecodeParams &p, const SegPlan &plan) {
  using C = typename W::C;
  using T = typename W::Elem_;
  constexpr int D = C::D, kVecs = C::kHeads * D / 4;
  constexpr int kPer = (kVecs + kJoinLanes - 1) / kJoinLanes;
  constexpr int kBatches = kMaxCtas / 32;
  constexpr float kNone = -1.f;  // the share of a part without keys, whose sums are not read
  static_assert(C::kHeads <= kJoinLanes * kJoinWays / 32, "a warp to a query head");
  __shared__ float4 sums[kJoinWays][kVecs];
  __shared__ float share[kMaxCtas][C::kHeads];
  const int ctas = gridDim.x, first = blockIdx.x;
  const int lane = threadIdx.x % kJoinLanes, way = threadIdx.x / kJoinLanes;
  const int head = threadIdx.x / 32, part = threadIdx.x % 32;
  const float *base = p.workspace + static_cast<int64_t>(first) * 2 * C::kState;
  auto state_of = [&](int k) {  // the first CTA's second state, then the others' first
    return base + (k == 0 ? 1 : 2 * k) * C::kState;
  };
  auto read = [&](int k, float4 (&a)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = lane + i * kJoinLanes;
      if (v < kVecs) a[i] = __ldcg(reinterpret_cast<const float4 *>(state_of(k)) + v);
    }
  };
  pdl_wait();
  pdl_launch_dependents();
  const SegMeta meta =
      reinterpret_cast<const SegMeta *>(p.workspace + static_cast<int64_t>(ctas) * 2 * C::kState)[first];
  float4 x[kPer];
  if (first + way < ctas) read(way, x);
  if (meta.segment < 0) return;
  const int parts = min(meta.parts, ctas - first);
  if (head < C::kHeads) {
    float m[kBatches], l[kBatches], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
      m[i] = -INFINITY, l[i] = 0.f;
      if (i * 32 + part >= parts) continue;
      const float *st = state_of(i * 32 + part) + C::kHeads * D + head;
      m[i] = __ldcg(st), l[i] = __ldcg(st + C::kHeads);
      M = fmaxf(M, m[i]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, off));
#pragma unroll
    for (int i = 0; i < kBatches; ++i) L += part_factor(m[i], l[i], M) * l[i];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(kAll, L, off);
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
      if (i * 32 + part >= parts) break;
      const bool none = m[i] == -INFINITY && l[i] == 0.f;
      share[i * 32 + part][head] = none ? kNone : L == 0.f ? 0.f : __fdividef(part_factor(m[i], l[i], M) * l[i], L);
    }
  }
  __syncthreads();
  float4 A[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) A[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = way; k < parts; k += kJoinWays) {
    float4 y[kPer];
    if (k + kJoinWays < parts) read(k + kJoinWays, y);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = lane + i * kJoinLanes;
      if (v >= kVecs) break;
      const float s = share[k][v * 4 / D];
      if (s == kNone) continue;
      A[i].x = fmaf(s, x[i].x, A[i].x), A[i].y = fmaf(s, x[i].y, A[i].y);
      A[i].z = fmaf(s, x[i].z, A[i].z), A[i].w = fmaf(s, x[i].w, A[i].w);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = y[i];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = lane + i * kJoinLanes;
    if (v < kVecs) sums[way][v] = A[i];
  }
  __syncthreads();
  const int G = p.num_q_heads / p.num_kv_heads, H = p.num_kv_heads * plan.tiles;
  const int s = static_cast<int>(plan.by_segments.div(meta.segment)), ht = meta.segment - s * H;
  const int kvh = static_cast<int>(plan.by_tiles.div(ht)), h0 = (ht - kvh * plan.tiles) * C::kHeads;
  const int heads = min(C::kHeads, G - h0);
  T *out = static_cast<T *>(p.out) + (static_cast<int64_t>(s) * p.num_q_heads + kvh * G + h0) * D;
  for (int e = threadIdx.x; e < heads * D; e += kJoinLanes * kJoinWays) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWays; ++w) a += reinterpret_cast<const float *>(sums[w])[e];
    out[e] = Elem<T>::from_float(a);
  }
}

template <class W>
cudaError_t launch_segments(void (*kern)(CodedDecodeParams, SegPlan), void (*join_kern)(CodedDecodeParams, SegPlan),
                            const CodedDecodeParams &p, int tiles, bool join, int ctas, cudaStream_t stream) {
  using C = typename W::C;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  const SegPlan plan = {tiles, FastDiv(p.num_kv_heads * tiles), FastDiv(tiles), FastDiv(p.block_size / kSegGroup),
                        FastDiv(ctas)};
  cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(C::kWarps * 32), C::kSmem, stream, p, plan);
  if (e == cudaSuccess && join)
    e = launch_pdl(join_kern, dim3(ctas), dim3(kJoinLanes * kJoinWays), 0, stream, p, plan);
  return e;
}

int segment_ctas(int sms) { return sms < kMaxCtas ? sms : kMaxCtas; }

// Whether some lengths that the table can hold need the second launch: not when
// every segment has a CTA and a full table is no more than `aligned` units.
bool segments_join(int64_t segments, int64_t capacity, int aligned, int sms) {
  return segments > sms || capacity > static_cast<int64_t>(aligned) * kUnit;
}

size_t segment_workspace(int heads, int head_dim, int sms) {
  return static_cast<size_t>(sms) * (2 * static_cast<size_t>(heads) * (head_dim + 2) * sizeof(float) + sizeof(SegMeta));
}

// 32-bit unit and group counts: more than any memory holds, or a table of more than 2^31 units a sequence.
bool segments_supported(int64_t segments_of_sequence, int num_kv_heads, int64_t num_blocks, int block_size,
                        int64_t capacity) {
  return num_blocks < (int64_t{1} << 31) / num_kv_heads / (block_size / kSegGroup) &&
         capacity / kUnit + 1 < (int64_t{1} << 31) / segments_of_sequence;
}

// `one(p)` for slices of the sequences whose units stay in 32 bits and whose prefix sums fit.
template <typename F>
cudaError_t launch_segment_slices(const CodedDecodeParams &p, int tiles, int dtype, F one) {
  const int64_t capacity = p.bt_stride * p.block_size;
  const int64_t H = static_cast<int64_t>(p.num_kv_heads) * tiles;
  int64_t slice = ((int64_t{1} << 31) - 1) / ((capacity / kUnit + 1) * H);
  if (slice > kMaxSeqs) slice = kMaxSeqs;
  for (int64_t s = 0; s < p.num_seqs; s += slice) {
    CodedDecodeParams q = p;
    q.num_seqs = p.num_seqs - s < slice ? p.num_seqs - s : slice;
    const int64_t row = s * p.num_q_heads * p.head_dim * (dtype == MI_DTYPE_FLOAT32 ? 4 : 2);
    q.query = static_cast<const char *>(p.query) + row;
    q.out = static_cast<char *>(p.out) + row;
    q.block_tables = p.block_tables + s * p.bt_stride;
    q.context_lens = p.context_lens + s;
    const cudaError_t e = one(q);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

}  // namespace mi
