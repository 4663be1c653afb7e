// Causal chunked prefill straight from the 8-bit cache (layout: fp8.cuh) on tcgen05, for 16-bit queries of head_dim 64 and
// 128 and any GQA group.
//
// Codes are exact in f16 and a group of 16 keys has one scale, so K and V go into the tensor cores as f16 without
// their scales: no rows are gathered, and 256 query rows share what is decoded once.  K's scale joins the factor that 16 scores
// of a row meet on their way into the exponential, V's joins the exponent of the same 16 p, which costs the softmax a
// multiplication and an addition per 16 keys.  q rows are multiplied by a power of two that puts their largest
// element into [2^14, 2^15) and converted to f16; O is held in units of 2^(R - 127), R at or above V's scale bytes.
//
// Unit of work: a pair of 128-row query tiles of one sequence and kv head, a row being (token, query head of the group), against
// the keys that it sees, 128 at a time.  The units' tiles, weighted by what they take, are one list that is cut into
// equal ranges, one per CTA (one to an SM), so ragged batches, a single long chunk and a few rows over a long context
// load every SM alike; a unit that is cut leaves its parts as means of V with their m and l, which a second launch joins.
//
// Roles (512 threads; registers are dealt out anew between them):
//   warps 0-3, 4-7   softmax of tile A and of tile B: one TMEM lane (row) a thread; then, while
//                    the last P V is under way, the next item's row of q, and the rows of this one
//   warps 8-11       decode K and V tiles, one conversion for two codes, into the 128-byte-swizzled layout that the MMA reads
//   warps 12, 15     issue the MMAs of tile A and of tile B, P V of a key tile, then S of the next: one thread for both is busy
//                    4600 cycles a tile with issuing and with the stalls of its waits, and everything else waits for it
//   warp 13          walks the work list and tells the others of each item, looks up pages and scales ahead and brings the
//                    codes of a tile by bulk copies
//   warp 14          looks for NaN of V in groups of scale 0
// TMEM: S_A at 0, S_B at 128, O_A at 256, O_B at 384; P (f16 pairs) goes over the first 64 columns of its S and is the A
// operand of P V from there.  Barriers and rings stay up across items; each role counts their phases.
// Every wait is bounded; a timeout flags MI_DEV_TIMEOUT, unwinds every role, waits for the MMAs, frees TMEM and returns.
//
// What it leaves to the kernel on the warp-level tensor cores, launched behind it for those sequences and heads alone ("odd"): a NaN
// of V (0 * NaN reaches rows that do not see its key), scales of V more than 14 binades below R, which is at most 2 above the largest
// that the item has met so far and never falls, scores past 2^20 or whose factor leaves fp32's range.  Without any it returns at once.
//
// Measured (cold L2): head_dim 64, 32 heads on 8: 1 x 256 rows on 16000 keys 110 us, 1 x 2048 on 6144 316 us (380 TFLOP/s; the warp-level
// kernel 698), 4 x 1024 on 4000 320; 6 x 300 87 us; head_dim 128: 1 x 128 on 16000 95 us (194 there), 12 heads
// on 2, 1 x 4096 155 us (376 there).  A pair of tiles over 128 keys takes 6000 cycles, of which a row's thread waits 2450 for S, spends
// 2400 on the exponentials and 900 on the maximum; the MMAs are 1024, the special functions of both tiles 2048.  Not what holds it: decoding
// (the same without), spinning waits, the factors of the scales, both tiles in step (taking turns: 502 to 512 us).
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.cuh"
#include "params.cuh"
#include "prefill_fp8.cuh"
#include "tc_helpers.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 512, kDecoders = 128;
constexpr int kHalf = 16384;  // 128 rows x 128 bytes
constexpr int kVStages = 2;
// Ring of scales: the entry of a tile is written when its codes are asked for: after the tile before it was decoded, so S of the one
// kKStages before that is done and P of the one before that stored, whose entry was the last to be read: kKStages + 2 entries.
constexpr int kItems = 4;  // items ahead
constexpr int kFactorMax = 94;             // largest exponent of a score's factor: sums of products are below 2^32
constexpr float kLift = 11.f, kLag = 4.f;  // p is 2^(x - m + kLift), m this far behind at most: within f16
constexpr int kSpread = 14;                // binades below R that p takes in
constexpr float kExact = 0x1p20f;          // m up to here is off by 2^-4 at most

template <int D>
struct TcCfg {
  static constexpr int kKStages = D == 64 ? 3 : 2;  // K is released early, after S
  static constexpr int kTile = D / 64 * kHalf;      // 128 rows of f16
  static constexpr int kGroup = f8_group_bytes(D);
  static constexpr int kRaw = 8 * kGroup;           // codes of a tile of K or V
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + 2 * kTile;
  static constexpr int kOffV = kOffK + kKStages * kTile;
  static constexpr int kOffRaw = kOffV + kVStages * kTile;
  static constexpr int kOffMisc = kOffRaw + 2 * kRaw;
  static constexpr int kScaleRing = kKStages + 2;
  static constexpr int kOffScales = kOffMisc + 288;
  static constexpr int kOffItems = kOffScales + 32 * kScaleRing;
  static constexpr int kSmem = kOffItems + kItems * static_cast<int>(sizeof(F8Item)) + 1024;
  static constexpr int kPer = 128 * D / 16 / kDecoders;  // 16-byte chunks of a tile per decoding thread
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
  static_assert((kKStages + kVStages) * kTile >= (kF8MaxSeqs + 1 + 32) * 8, "the prefix sums lie in the rings at the start");
};

enum {
  B_QFULL = 0,    // +tile: q of the item in shared memory (128 threads, which have seen the last S of the one before)
  B_KFULL = 2,    // +stage (the decoding threads)
  B_KEMPTY = 5,   // +stage (both issuers)
  B_VFULL = 8,    // +stage (the decoding threads)
  B_VEMPTY = 10,  // +stage (both issuers)
  B_SFULL = 12,   // +tile: S_X(j), and everything issued before it, done
  B_PFULL = 14,   // +tile: P_X(j) in TMEM (128 threads)
  B_ODONE = 16,   // +tile: the item's O_X final
  B_OEMPTY = 18,  // +tile: the item's O_X read (128 threads)
  B_RAWFULL = 20,   // +operand: codes of a tile landed
  B_RAWEMPTY = 22,  // +operand: decoded (the decoding threads)
  B_ITEMFULL = 24,   // +slot
  B_ITEMEMPTY = 28,  // +slot (softmax threads and issuer)
  B_FIN = 32,
  B_INFO = 33,    // two words: what the loader says of the tile of K and of V
  B_COUNT = 34
};
static_assert(B_COUNT * 8 + 16 <= 288 && kItems == 4, "their place in shared memory");
constexpr uint32_t kNoMore = 1u << 31;  // of K's word: there is no tile; else bits 0-7 the groups that exist, 8-15 those whose
                                        // V is zero, 16-20 the keys of the last group that exists

__device__ __forceinline__ bool aborted(const int *flag) { return *(volatile const int *)flag != 0; }

template <int REGS>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
// 512 threads at 128 registers: what the roles hold after the exchange
constexpr int kSoftmaxRegs = 184, kDecodeRegs = 64, kIssueRegs = 80;
static_assert(2 * kSoftmaxRegs + kDecodeRegs + kIssueRegs == 4 * 128, "the registers of the launch");

__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2i(int e) {
  const int a = max(-126, min(127, e)), b = max(-126, min(127, e - a));
  return __uint_as_float(static_cast<uint32_t>(a + 127) << 23) * __uint_as_float(static_cast<uint32_t>(b + 127) << 23);
}
__device__ __forceinline__ int byte_of(uint32_t w, int i) { return static_cast<int>(w >> (8 * i) & 255u); }
__device__ __forceinline__ int largest_byte(uint32_t a, uint32_t b) {
  uint32_t t = __vmaxu4(a, b);
  t = __vmaxu4(t, t >> 16);
  return static_cast<int>(max(t & 255u, t >> 8 & 255u));
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_prefill_tc_kernel(const __grid_constant__ CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page,
                          const __grid_constant__ F8Scale scale) {
  using C = TcCfg<D>;
  constexpr int kKStages = C::kKStages;
  constexpr uint32_t kIdescQK = tc::idesc_f16(128, 128, 0, false);
  constexpr uint32_t kIdescPV = tc::idesc_f16(128, D, 0, true);
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *bar = reinterpret_cast<uint64_t *>(smem + C::kOffMisc);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar + B_COUNT);
  int *abort_flag = reinterpret_cast<int *>(tmem_slot + 1), *nan_flag = abort_flag + 1, *zero_flag = nan_flag + 1;
  constexpr int kScaleRing = C::kScaleRing;
  uint8_t *scales = smem + C::kOffScales;  // ring: K's bytes of 8 groups, V's, then a bit for each whose page is none
  F8Item *item_ring = reinterpret_cast<F8Item *>(smem + C::kOffItems);
  volatile uint32_t *info = reinterpret_cast<volatile uint32_t *>(bar + B_INFO);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) mbar_init(&bar[B_KFULL + s], kDecoders), mbar_init(&bar[B_KEMPTY + s], 2);
    for (int s = 0; s < kVStages; ++s) mbar_init(&bar[B_VFULL + s], kDecoders), mbar_init(&bar[B_VEMPTY + s], 2);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bar[B_QFULL + x], 128);
      mbar_init(&bar[B_SFULL + x], 1);
      mbar_init(&bar[B_PFULL + x], 128);
      mbar_init(&bar[B_ODONE + x], 1);
      mbar_init(&bar[B_OEMPTY + x], 128);
    }
    for (int o = 0; o < 2; ++o) mbar_init(&bar[B_RAWFULL + o], 1), mbar_init(&bar[B_RAWEMPTY + o], kDecoders);
    for (int i = 0; i < kItems; ++i) mbar_init(&bar[B_ITEMFULL + i], 1), mbar_init(&bar[B_ITEMEMPTY + i], 256 + 2);
    mbar_init(&bar[B_FIN], 2);
    *abort_flag = *nan_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) tc::tmem_alloc(tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  pdl_wait();
  int64_t *prefix = reinterpret_cast<int64_t *>(smem + C::kOffK);
  const F8Work work = f8_work(p, by_group, prefix, prefix + kF8MaxSeqs + 1, gridDim.x);
  F8Walker walk;
  if (warp == 13 || warp == 14) walk.start(p, by_group, prefix, work, blockIdx.x);
  __syncthreads();  // the prefix sums are read: the rings are free
  // Item i, or null where there is none (or something has gone wrong: !ok).
  auto item = [&](uint32_t i, bool &ok) -> const F8Item * {
    ok = mbar_wait_bounded(&bar[B_ITEMFULL + i % kItems], i / kItems & 1, p.status) && !aborted(abort_flag);
    const F8Item *it = item_ring + i % kItems;
    return ok && it->kvh >= 0 ? it : nullptr;
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    more_registers<kSoftmaxRegs>();
    const int x = warp >> 2, r = threadIdx.x & 127;  // query tile, TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + x * 128 + lane_off, tO = tmem + 256 + x * 128 + lane_off;
    const int G = p.num_q_heads / p.num_kv_heads;
    uint32_t sc = 0, uses = 0, tiles = 0;
    bool ok = true, odd = false;
    F8Meta meta = {0, 0, 0, 0};
    auto get = [&](uint32_t number) {
      bool good;
      const F8Item *it = item(number, good);
      ok = __all_sync(kAll, good);
      return ok ? it : nullptr;
    };
    // This thread's row of q as f16 in shared memory; returns the exponent that its products want, without K's scale.
    auto load_q = [&](const F8Item *it) -> int {
      if (it == nullptr || it->end[x] <= it->j0) return 0;
      const uint32_t row = static_cast<uint32_t>(it->row0) + x * 128 + r, at = by_group.div(row);
      const int64_t token = static_cast<int64_t>(it->q0) + at;
      const bool there = r < it->rows[x] && token >= 0 && token < p.num_tokens;
      uint4 raw[D / 8];
      const uint4 *from = reinterpret_cast<const uint4 *>(
          static_cast<const T *>(p.query) + (token * p.num_q_heads + it->kvh * G + (row - at * G)) * D);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (there) raw[i] = __ldg(from + i);
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {  // bits order like the values, two to a word
        const uint32_t a = __vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), b = __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu);
        top = __vmaxu2(top, __vmaxu2(a, b));
      }
      const uint16_t most = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
      top = __float_as_uint(Elem<T>::to_float(*reinterpret_cast<const T *>(&most)));
      // not finite: as it is; nor do zeros need a power
      const int e = top >= 0x7f800000u || top == 0 || scale.sign == 0.f ? 0 : min(14 - (static_cast<int>(top >> 23) - 127), 126);
      const float f = exp2i(e) * scale.sign;
      uint8_t *to = smem + C::kOffQ + x * C::kTile + r * 128;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        float2 v[4];
        Vec16<T>::unpack(raw[c], v);
        *reinterpret_cast<uint4 *>(to + (c >> 3) * kHalf + (((c & 7) ^ (r & 7)) << 4)) =
            make_uint4(pack16(v[0].x * f, v[0].y * f), pack16(v[1].x * f, v[1].y * f), pack16(v[2].x * f, v[2].y * f),
                       pack16(v[3].x * f, v[3].y * f));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bar[B_QFULL + x]);
      return scale.exponent - e;
    };
    const F8Item *it = get(0);
    int power = load_q(it);
    for (uint32_t number = 0; ok && it != nullptr; ++number) {
      const int j0 = it->j0, jend = it->end[x];
      const bool used = jend > j0;
      const bool valid = r < it->rows[x];
      const int seen = valid ? max(0, min(it->prefix + static_cast<int>(by_group.div(static_cast<uint32_t>(it->row0 + x * 128 + r))) + 1,
                                          it->keys))
                             : 0;  // keys
      float m = -INFINITY, l = 0.f, unit = 0.f;
      int ref = -1, top_byte = -1;
      for (int j = j0; j < jend; ++j) {
        if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_SFULL + x], sc & 1, p.status) && !aborted(abort_flag))) {
          ok = false;
          break;
        }
        ++sc;
        tc::fence_after_sync();
        // The whole row in registers, one TMEM round trip per tile (read twice in pieces it takes half as many registers
        // and 549 us where this takes 512, 1536 on 12288: a round trip beside the MMAs is some 250 cycles).
        float sr[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tc::tmem_ld32(tS + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) sr[c * 32 + i] = v[i];
        }
        const uint8_t *entry = scales + (tiles + (j - j0)) % kScaleRing * 32;
        const uint4 sb = *reinterpret_cast<const uint4 *>(entry);
        const uint32_t none = *reinterpret_cast<const uint32_t *>(entry + 16);
        if (j == j0) {
          const bool normal = power >= -126 && power <= kFactorMax;
          unit = __uint_as_float(static_cast<uint32_t>((normal ? power : 0) + 127) << 23) * scale.mantissa;
          top_byte = normal ? kFactorMax + 127 - power : -1;
        }
        tc::tmem_wait_ld();
        odd |= valid && largest_byte(sb.x, sb.y) > top_byte;
        // key c of the tile is visible iff c < seen - 128 j: only diagonal tiles (and rows past the chunk) mask anything
        const int lim = seen - j * 128;
        if (lim < 128) {
#pragma unroll
          for (int c = 0; c < 128; ++c) sr[c] = c < lim ? sr[c] : -INFINITY;
        }
        if (none) {  // groups without a page; uniform
#pragma unroll
          for (int c = 0; c < 128; ++c) sr[c] = none >> (c / 16) & 1u ? -INFINITY : sr[c];
        }
        // K's scale of a group times the row's unit; not 0, which a masked score would make a NaN
        auto factor = [&](int q) {
          return fmaxf(f8_scale(static_cast<uint32_t>(byte_of(q < 4 ? sb.x : sb.y, q & 3))) * unit, 0x1p-126f);
        };
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float a = fmax3(sr[16 * q], sr[16 * q + 1], sr[16 * q + 2]), b = fmax3(sr[16 * q + 3], sr[16 * q + 4], sr[16 * q + 5]);
#pragma unroll
          for (int i = 6; i < 14; i += 4) {
            a = fmax3(a, sr[16 * q + i], sr[16 * q + i + 1]);
            b = fmax3(b, sr[16 * q + i + 2], sr[16 * q + i + 3]);
          }
          a = fmax3(a, sr[16 * q + 14], sr[16 * q + 15]);
          mx = fmaxf(mx, fmaxf(a, b) * factor(q));
        }
        float m_new = m, alpha = 1.f, turn = 1.f;  // turn: what O is multiplied by
        if (mx > m + kLag) {
          m_new = mx;
          alpha = m != -INFINITY ? fast_exp2(m - m_new) : 0.f;
          turn = alpha;
        }
        const int v_top = largest_byte(sb.z, sb.w);
        if (v_top > ref) {  // uniform in the tile
          const int next = v_top + 2;  // two binades of room
          if (ref >= 0) turn *= exp2i(ref - next);
          ref = next;
        }
        odd |= fabsf(m_new) > kExact && m_new != -INFINITY;
        // P = 2^(s * factor - m + kLift + V's byte - R) as f16 pairs over the first 64 columns of S
        const float nb = m_new == -INFINITY ? 0.f : kLift - m_new;  // masked: 2^-inf = 0
        float sum = 0.f;
        int lowest = 0;
#pragma unroll
        for (int h = 0; h < 4; ++h) {  // keys 32h .. 32h + 31 -> columns 16h .. 16h + 15
          float pk[16];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int q = 2 * h + i, vb = byte_of(q < 4 ? sb.z : sb.w, q & 3);
            const int below = vb == 0 ? 0 : max(vb - ref, -100);  // of scale 0: decoded to zeros
            lowest = min(lowest, below);
            const float f = factor(q), nq = nb + static_cast<float>(below);
            const float2 f2 = make_float2(f, f), n2 = make_float2(nq, nq);
            float2 part = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 a2 = ffma2(make_float2(sr[16 * q + 2 * k], sr[16 * q + 2 * k + 1]), f2, n2);
              const float2 e = make_float2(fast_exp2(a2.x), fast_exp2(a2.y));
              part = fadd2(part, e);
              pk[8 * i + k] = __uint_as_float(pack16(e.x, e.y));
            }
            sum = fmaf(part.x + part.y, __uint_as_float(static_cast<uint32_t>(127 - below) << 23), sum);
          }
          tc::tmem_st16(tS + h * 16, pk);
        }
        odd |= lowest < -kSpread;
        // O_X is quiescent here (PV_X(j-1) completed before S_X(j) did) and PV_X(j) waits for this thread's arrival below
        if (j > j0 && __any_sync(kAll, turn != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tc::tmem_ld32(tO + c * 32, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= turn;
            tc::tmem_st32(tO + c * 32, o);
          }
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        mbar_arrive(&bar[B_PFULL + x]);
        l = fmaf(l, alpha, sum);
        m = m_new;
      }
      if (!ok) break;
      const F8Item *next = get(number + 1);
      if (!ok) break;
      power = load_q(next);
      if (used) {
        ok = __all_sync(kAll, mbar_wait_bounded(&bar[B_ODONE + x], uses & 1, p.status) && !aborted(abort_flag));
        if (!ok) break;
        tc::fence_after_sync();
      }
      const float inv = l == 0.f ? 0.f : 1.f / l, back = exp2i(ref - 127);
      const bool whole = it->first && it->last;
      const uint32_t row = static_cast<uint32_t>(it->row0) + x * 128 + r, at = by_group.div(row);
      const int64_t token = static_cast<int64_t>(it->q0) + at;
      const bool stored = valid && token >= 0 && token < p.num_tokens;
      if (valid && !stored) flag_status(p.status, MI_DEV_BAD_SLOT);
      T *orow = static_cast<T *>(p.out) + (token * p.num_q_heads + it->kvh * G + (row - at * G)) * D;
      // a part: m, l and the mean of V, each [256 rows], so that a warp's stores are whole lines
      float *state = p.workspace + (static_cast<int64_t>(blockIdx.x) * 2 + (it->first ? 1 : 0)) * 256 * (D + 2) + x * 128 + r;
      if (!whole && valid) state[0] = m, state[256] = l;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (used) {
          tc::tmem_ld32(tO + c * 32, o);
          tc::tmem_wait_ld();
        } else {  // no visible key
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o[i] = o[i] * inv * back;
          odd |= valid && o[i] != o[i];  // a NaN, wherever it comes from
        }
        if (whole && stored) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = Elem<T>::from_float(o[i + k]);
            *reinterpret_cast<uint4 *>(orow + c * 32 + i) = w;
          }
        } else if (!whole && valid) {
#pragma unroll
          for (int i = 0; i < 32; ++i) state[(2 + c * 32 + i) * 256] = o[i];
        }
      }
      if (used) {  // O_X is read: the next item's first P V may overwrite it
        tc::fence_before_sync();
        mbar_arrive(&bar[B_OEMPTY + x]);
        ++uses;
      }
      if (it->first && !it->last) meta = {it->seq, it->kvh, it->pair, it->parts};
      tiles += it->j1 - j0;
      mbar_arrive(&bar[B_ITEMEMPTY + number % kItems]);
      it = next;
    }
    if (!ok && lane == 0) *(volatile int *)abort_flag = 1;
    const bool any = __any_sync(kAll, odd);
    if (lane == 0) f8_odd(p, D, gridDim.x)[blockIdx.x * 8 + warp] = any;
    if (threadIdx.x == 0) f8_meta(p, D, gridDim.x)[blockIdx.x] = meta;
  } else if (warp < 12) {
    // ------------------------------------------------------------ decode
    fewer_registers<kDecodeRegs>();
    const int tid = threadIdx.x - 256;
    const uint8_t *raw_k = smem + C::kOffRaw, *raw_v = raw_k + C::kRaw;
    bool ok = true;
    for (uint32_t t = 0;; ++t) {
      const uint32_t ks = t % kKStages, vs = t % kVStages;
      if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_RAWFULL], t & 1, p.status) && !aborted(abort_flag))) {
        ok = false;
        break;
      }
      if (info[0] & kNoMore) break;
      if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_KEMPTY + ks], (t / kKStages & 1) ^ 1, p.status) && !aborted(abort_flag))) {
        ok = false;
        break;
      }
      uint8_t *to = smem + C::kOffK + ks * C::kTile;
#pragma unroll 4
      for (int n = 0; n < C::kPer; ++n) {  // 16 dims of a key; of groups that do not exist whatever lies there, all masked
        const int id = n * kDecoders + tid, group = id / D, i = id % D % 64, part = id % D / 64;
        const int key = group * kF8Group + i / 4, c = i % 4 * 2;
        const uint4 w = *reinterpret_cast<const uint4 *>(raw_k + group * C::kGroup + id % D * 16);
        uint32_t h[8];
        f8_to_f16(w.x, h[0], h[1]);
        f8_to_f16(w.y, h[2], h[3]);
        f8_to_f16(w.z, h[4], h[5]);
        f8_to_f16(w.w, h[6], h[7]);
        uint8_t *row = to + part * kHalf + key * 128;
        *reinterpret_cast<uint4 *>(row + ((c ^ (key & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(row + (((c + 1) ^ (key & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      mbar_arrive(&bar[B_RAWEMPTY]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bar[B_KFULL + ks]);
      if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_RAWFULL + 1], t & 1, p.status) &&
                                mbar_wait_bounded(&bar[B_VEMPTY + vs], (t / kVStages & 1) ^ 1, p.status) && !aborted(abort_flag))) {
        ok = false;
        break;
      }
      const uint32_t says = info[1], there = says & 255u & ~(says >> 8);  // groups with values
      const int last = 31 - __clz(static_cast<int>(says & 255u)), in_last = static_cast<int>(says >> 16 & 31u);
      to = smem + C::kOffV + vs * C::kTile;
#pragma unroll 4
      for (int n = 0; n < C::kPer; ++n) {  // 8 dims of a pair of keys
        const int id = n * kDecoders + tid, group = id / D, i = id % D % 64, part = id % D / 64;
        const int tok = i / 32 * 8 + i % 4 * 2, key = group * kF8Group + tok, c = i % 32 / 4;
        uint4 w = *reinterpret_cast<const uint4 *>(raw_v + group * C::kGroup + id % D * 16);
        if (!(there >> group & 1u)) w = make_uint4(0u, 0u, 0u, 0u);
        if (group == last && in_last < kF8Group) {  // past the context anything may lie
          const uint32_t keep = (tok < in_last ? 0x00ff00ffu : 0u) | (tok + 1 < in_last ? 0xff00ff00u : 0u);
          w = make_uint4(w.x & keep, w.y & keep, w.z & keep, w.w & keep);
        }
        uint32_t h[8];  // pairs of keys, dim after dim
        f8_to_f16(w.x, h[0], h[1]);
        f8_to_f16(w.y, h[2], h[3]);
        f8_to_f16(w.z, h[4], h[5]);
        f8_to_f16(w.w, h[6], h[7]);
        uint8_t *row = to + part * kHalf + key * 128;
        *reinterpret_cast<uint4 *>(row + ((c ^ (key & 7)) << 4)) =
            make_uint4(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410), __byte_perm(h[4], h[5], 0x5410),
                       __byte_perm(h[6], h[7], 0x5410));
        *reinterpret_cast<uint4 *>(row + 128 + ((c ^ (key + 1 & 7)) << 4)) =
            make_uint4(__byte_perm(h[0], h[1], 0x7632), __byte_perm(h[2], h[3], 0x7632), __byte_perm(h[4], h[5], 0x7632),
                       __byte_perm(h[6], h[7], 0x7632));
      }
      mbar_arrive(&bar[B_RAWEMPTY + 1]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bar[B_VFULL + vs]);
    }
    if (!ok && lane == 0) *(volatile int *)abort_flag = 1;
  } else {
    fewer_registers<kIssueRegs>();
    if (warp == 12 || warp == 15) {
      // ---------------------------------------------------------- MMA issuers, one to a query tile
      if (lane == 0) {
        const int x = warp == 12 ? 0 : 1;
        const uint32_t tS = tmem + x * 128, tO = tmem + 256 + x * 128;
        uint32_t t = 0, sc = 0, uses = 0;  // K and V tiles passed, S products issued, items that used this tile
        bool ok = true;
        // Descriptors: a K step or a ring slot moves the start address field of the low word (16-byte units), the high word stays.
        const uint32_t qd = static_cast<uint32_t>(tc::smem_desc_sw128(smem_addr(smem + C::kOffQ + x * C::kTile), 16, 1024));
        const uint32_t kd0 = static_cast<uint32_t>(tc::smem_desc_sw128(smem_addr(smem + C::kOffK), 16, 1024));
        const uint32_t vd0 = static_cast<uint32_t>(tc::smem_desc_sw128(smem_addr(smem + C::kOffV), kHalf, 1024));
        const uint32_t high = static_cast<uint32_t>(tc::smem_desc_sw128(0, 16, 1024) >> 32);
        auto desc = [&](uint32_t low) { return static_cast<uint64_t>(high) << 32 | low; };
        constexpr uint32_t kTile16 = C::kTile >> 4;
        auto kstep = [](int kk) -> uint32_t { return static_cast<uint32_t>(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4); };
        auto full = [&](int which, uint32_t stages, uint32_t at) {
          return mbar_spin_bounded(&bar[which + at % stages], at / stages & 1, p.status);
        };
        auto s_mma = [&](uint32_t at) {  // S = Q K^T with the K tile at ring position `at`
          const uint32_t kd = kd0 + at % kKStages * kTile16;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            tc::umma_f16(tS, desc(qd + kstep(kk)), desc(kd + kstep(kk)), kIdescQK, kk > 0 ? 1u : 0u);
          tc::umma_commit(&bar[B_SFULL + x]);
          tc::umma_commit(&bar[B_KEMPTY + at % kKStages]);
          ++sc;
        };
        for (uint32_t number = 0;; ++number) {
          const F8Item *it = item(number, ok);
          if (it == nullptr) break;
          const int j0 = it->j0, j1 = it->j1, end = it->end[x];
          mbar_arrive(&bar[B_ITEMEMPTY + number % kItems]);
          if (end > j0) {
            ok = mbar_spin_bounded(&bar[B_QFULL + x], uses & 1, p.status) && full(B_KFULL, kKStages, t) && !aborted(abort_flag);
            if (!ok) break;
            tc::fence_after_sync();
            s_mma(t);
          }
          for (int j = j0; j < j1; ++j, ++t) {
            // What is needed besides P is waited for before it: then the P V and the next S go out without a pause.
            const bool mine = j < end, more = j + 1 < end;
            if (!mine && j == j0) {  // not of this query tile: its slots are let go
              if (!(ok = full(B_KFULL, kKStages, t))) break;
              mbar_arrive(&bar[B_KEMPTY + t % kKStages]);
            }
            ok = full(B_VFULL, kVStages, t) && (j + 1 >= j1 || full(B_KFULL, kKStages, t + 1)) && !aborted(abort_flag);
            // The first P V overwrites O: the previous item's must be read out.
            if (ok && mine && j == j0) ok = mbar_spin_bounded(&bar[B_OEMPTY + x], (uses & 1) ^ 1, p.status);
            if (ok && mine) ok = mbar_spin_bounded(&bar[B_PFULL + x], (sc - 1) & 1, p.status);
            if (!ok) break;
            tc::fence_after_sync();
            if (mine) {
              const uint32_t vd = vd0 + t % kVStages * kTile16;
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)  // P from TMEM
                tc::umma_f16_tmem_a(tO, tS + kk * 8, desc(vd + kk * (2048 >> 4)), kIdescPV, (j > j0 || kk > 0) ? 1u : 0u);
              tc::umma_commit(&bar[B_VEMPTY + t % kVStages]);
            } else {
              mbar_arrive(&bar[B_VEMPTY + t % kVStages]);
            }
            if (more)
              s_mma(t + 1);
            else if (j + 1 < j1)
              mbar_arrive(&bar[B_KEMPTY + (t + 1) % kKStages]);
          }
          if (!ok) break;
          if (end > j0) {
            tc::umma_commit(&bar[B_ODONE + x]);
            ++uses;
          }
        }
        if (!ok) *(volatile int *)abort_flag = 1;
        tc::umma_commit(&bar[B_FIN]);  // every MMA completes before TMEM is released
        mbar_spin_bounded(&bar[B_FIN], 0, p.status);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ---------------------------------------------------------- loader
      const int per_page = p.block_size / kF8Group;
      uint8_t *raw = smem + C::kOffRaw;
      uint32_t tiles = 0;
      uint32_t number = 0;
      bool ok = true, told = false;
      // To warp 14, once: there is a group of V of scale 0, or there is none.
      auto tell_zero = [&](int is) {
        if (told) return;
        told = true;
        if (lane == 0) *(volatile int *)zero_flag = is;
        __syncwarp();
        asm volatile("bar.arrive 1, 64;" ::: "memory");
      };
      F8Item it;
      auto tell = [&] {  // the others of the item
        if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_ITEMEMPTY + number % kItems], (number / kItems & 1) ^ 1, p.status) &&
                                  !aborted(abort_flag)))
          return false;
        if (lane == 0) {
          item_ring[number % kItems] = it;
          mbar_arrive(&bar[B_ITEMFULL + number % kItems]);
        }
        ++number;
        return true;
      };
      while (walk.next(p, by_group, it)) {
        if (!(ok = tell())) break;
        if (it.j0 >= it.j1) continue;
        const int32_t *table = p.block_tables + it.seq * p.bt_stride;
        // A lane looks up a group of a tile (lanes 8 to 15 the same ones, for V's scales); -1 past the keys, -2: its page is none
        auto page_of = [&](int j) {
          const int group = j * 8 + (lane & 7);
          return group * kF8Group < it.keys && j < it.j1 ? __ldg(table + by_page.div(group)) : INT32_MIN;
        };
        auto place_of = [&](int j, int page) {
          const int group = j * 8 + (lane & 7);
          if (group * kF8Group >= it.keys || j >= it.j1) return -1;
          if (page < 0 || page >= p.num_blocks) return -2;
          return (page * p.num_kv_heads + it.kvh) * per_page + group - static_cast<int>(by_page.div(group)) * per_page;
        };
        auto scale_of = [&](int place) {
          const uint8_t *pool = lane < 8 ? p.key_pages : p.value_pages;
          return place >= 0 && lane < 16 ? static_cast<uint32_t>(pool[static_cast<int64_t>(place) * C::kGroup + kF8Group * D]) : 0u;
        };
        int place = place_of(it.j0, page_of(it.j0)), ahead = page_of(it.j0 + 1);
        uint32_t byte = scale_of(place);
        for (int j = it.j0; j < it.j1; ++j, ++tiles) {
          const int next = place_of(j + 1, ahead);
          ahead = page_of(j + 2);
          const uint32_t next_byte = scale_of(next);
          const unsigned exists = __ballot_sync(kAll, lane < 8 && place >= 0), none = __ballot_sync(kAll, lane < 8 && place == -2);
          const unsigned zero = __ballot_sync(kAll, lane >= 8 && lane < 16 && byte == 0) >> 8;
          if (zero & exists) tell_zero(1);
          // keys of the last group that exists (later ones may have no page; theirs are zeros in any case)
          const int last = 31 - __clz(static_cast<int>(exists));
          const int in_last = exists ? min(kF8Group, it.keys - (j * 8 + last) * kF8Group) : 0;
#pragma unroll
          for (int o = 0; o < 2; ++o) {  // K, V
            if (!__all_sync(kAll, mbar_wait_bounded(&bar[B_RAWEMPTY + o], (tiles & 1) ^ 1, p.status) && !aborted(abort_flag))) {
              ok = false;
              break;
            }
            if (o == 0) {
              uint8_t *entry = scales + tiles % kScaleRing * 32;
              if (lane < 16) entry[lane] = static_cast<uint8_t>(byte);
              if (lane == 16) *reinterpret_cast<uint32_t *>(entry + 16) = none;
              if (lane == 0 && none) flag_status(p.status, MI_DEV_BAD_BLOCK);
            }
            if (lane == 0) info[o] = exists | zero << 8 | static_cast<uint32_t>(in_last) << 16;
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&bar[B_RAWFULL + o], __popc(exists) * C::kGroup);
            __syncwarp();
            if (lane < 8 && place >= 0)
              bulk_g2s(raw + o * C::kRaw + lane * C::kGroup,
                       (o ? p.value_pages : p.key_pages) + static_cast<int64_t>(place) * C::kGroup, C::kGroup, &bar[B_RAWFULL + o]);
          }
          if (!ok) break;
          place = next, byte = next_byte;
        }
        if (!ok) break;
      }
      it.kvh = -1;
      if (ok) ok = tell();
      if (ok) ok = __all_sync(kAll, mbar_wait_bounded(&bar[B_RAWEMPTY], (tiles & 1) ^ 1, p.status) && !aborted(abort_flag));
      if (ok) {
        if (lane == 0) {
          info[0] = kNoMore;
          mbar_arrive(&bar[B_RAWFULL]);
        }
      } else if (lane == 0) {
        *(volatile int *)abort_flag = 1;
        // this CTA's own copies in flight land before its shared memory goes away
        for (int o = 0; o < 2; ++o)
          if (tiles > 0) mbar_wait_bounded(&bar[B_RAWFULL + o], (tiles - 1) & 1, p.status);
        mbar_wait_bounded(&bar[B_RAWFULL], tiles & 1, nullptr);  // the tile under way, if it was asked for
      }
      __syncwarp();
      tell_zero(0);
    } else {
      // ---------------------------------------------------------- NaN of V in groups of scale 0
      // Such groups are decoded to zeros; the store makes one with NaN codes of 16 tokens without a finite element but zeros.  This
      // warp goes over the CTA's keys by itself as soon as the loader has met one: in the decoding warps the look took 3 to 7 us of 75
      // (6 x 300 at head_dim 64, where there is none), in the loader up to 4%.
      asm volatile("bar.sync 1, 64;" ::: "memory");
      const int per_page = p.block_size / kF8Group;
      F8Item it;
      while (*(volatile const int *)zero_flag && walk.next(p, by_group, it)) {
        const int32_t *table = p.block_tables + it.seq * p.bt_stride;
        const int groups = min(it.j1 * 8, (it.keys + kF8Group - 1) / kF8Group);
        for (int g0 = it.j0 * 8; g0 < groups; g0 += 32) {
          const int group = g0 + lane, col = static_cast<int>(by_page.div(group));
          const int page = group < groups ? __ldg(table + col) : -1;
          const uint8_t *codes = p.value_pages;
          bool zero = page >= 0 && page < p.num_blocks;
          if (zero) {
            codes += static_cast<int64_t>((page * p.num_kv_heads + it.kvh) * per_page + group - col * per_page) * C::kGroup;
            zero = codes[kF8Group * D] == 0;
          }
          constexpr int kAtOnce = 256 / D;  // groups whose reads are on their way together
          for (unsigned left = __ballot_sync(kAll, zero); left;) {
            uint4 w[kAtOnce][D / 32];
            int tokens[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
              const int from = left ? __ffs(static_cast<int>(left)) - 1 : 0;
              const uint4 *at = reinterpret_cast<const uint4 *>(__shfl_sync(kAll, reinterpret_cast<unsigned long long>(codes), from));
              tokens[u] = left ? it.keys - (g0 + from) * kF8Group : 0;
#pragma unroll
              for (int i = 0; i < D / 32; ++i) w[u][i] = tokens[u] > 0 ? __ldg(at + i * 32 + lane) : make_uint4(0u, 0u, 0u, 0u);
              left &= left - 1;
            }
            bool nan = false;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
              for (int i = 0; i < D / 32; ++i) {
                const int tok = (i * 32 + lane) % 64 / 32 * 8 + lane % 4 * 2;  // 8 dims of it and the next
                const uint32_t keep = (tok < tokens[u] ? 0x00ff00ffu : 0u) | (tok + 1 < tokens[u] ? 0xff00ff00u : 0u);
                const uint4 v = w[u][i];
                nan |= f8_any_nan(v.x & keep) || f8_any_nan(v.y & keep) || f8_any_nan(v.z & keep) || f8_any_nan(v.w & keep);
              }
            if (nan) *(volatile int *)nan_flag = 1;
          }
        }
      }
    }
  }

  pdl_launch_dependents();
  tc::fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && *(volatile const int *)nan_flag) f8_odd(p, D, gridDim.x)[blockIdx.x * 8] = 1;
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Units that were cut: block (c, y) joins 32 rows of the one that goes on from CTA c, a lane to a row, a warp to an eighth of
// the dims.
template <typename T, int D>
__global__ void __launch_bounds__(256) fp8_prefill_tc_join_kernel(const CodedPrefillParams p, const FastDiv by_group, int ctas) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int N = D / 8;
  const int c = blockIdx.x, r = blockIdx.y * 32 + (threadIdx.x & 31), d0 = (threadIdx.x >> 5) * N;
  const F8Meta meta = f8_meta(p, D, ctas)[c];
  if (meta.parts == 0) return;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int64_t q0 = p.cu_seqlens_q[meta.seq];
  const int64_t row = static_cast<int64_t>(meta.pair) * 256 + r;
  if (row >= (p.cu_seqlens_q[meta.seq + 1] - q0) * G) return;
  const int64_t at = by_group.div(static_cast<uint32_t>(row)), token = q0 + at;
  if (token < 0 || token >= p.num_tokens) return;
  const int parts = min(meta.parts, ctas - c);
  float M = -INFINITY, L = 0.f, A[N];
#pragma unroll
  for (int i = 0; i < N; ++i) A[i] = 0.f;
#pragma unroll 2
  for (int k = 0; k < parts; ++k) {  // the first CTA's second state, then the others' first
    const float *st = p.workspace + (static_cast<int64_t>(c + k) * 2 + (k == 0)) * 256 * (D + 2) + r;
    const float m = __ldcg(st), l = __ldcg(st + 256);
    float a[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = __ldcg(st + (2 + d0 + i) * 256);
    if (m == -INFINITY && l == 0.f) continue;  // no keys
    const float next = fmaxf(M, m);
    const float f = M == -INFINITY ? (L == 0.f ? 0.f : 1.f) : fast_exp2(M - next);
    const float e = m == -INFINITY ? 1.f : fast_exp2(m - next);
    const float sum = f * L + e * l, share = sum == 0.f ? 0.f : e * l / sum;  // of this part in the mean
#pragma unroll
    for (int i = 0; i < N; ++i) A[i] = fmaf(share, a[i], A[i] - share * A[i]);
    L = sum;
    M = next;
  }
  T *out = static_cast<T *>(p.out) + (token * p.num_q_heads + static_cast<int64_t>(meta.kvh) * G + (row - at * G)) * D + d0;
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    uint4 w;
    T *e = reinterpret_cast<T *>(&w);
#pragma unroll
    for (int u = 0; u < 8; ++u) e[u] = Elem<T>::from_float(A[i + u]);
    reinterpret_cast<uint4 *>(out)[i / 8] = w;
  }
}

namespace {

template <typename T, int D>
cudaError_t launch_tc(const CodedPrefillParams &p, cudaStream_t stream) {
  using C = TcCfg<D>;
  auto kern = fp8_prefill_tc_kernel<T, D>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  const int ctas = sm_count_current();
  const FastDiv by_group(p.num_q_heads / p.num_kv_heads), by_page(p.block_size / kF8Group);
  cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(kThreads), C::kSmem, stream, p, by_group, by_page,
                             f8_softmax_scale(p.scale_log2));
  if (e == cudaSuccess)
    e = launch_pdl(fp8_prefill_tc_join_kernel<T, D>, dim3(ctas, 8), dim3(256), 0, stream, p, by_group, ctas);
  return e;
}

}  // namespace

// Whether this kernel takes a call, by its tiles of 128 rows x 128 keys (as many as the bounds allow): the one on the warp-level
// tensor cores (prefill_fp8.cu) starts in 12 us where this needs 32 to 44 (work list, the chain of look-ups, two launches
// behind it), but takes 2 to 3 times as long a tile.  Even at about 10 tiles an SM of head_dim 64 and 5 of 128, this : other in us:
// 1 x 64 rows on 64 keys 32 : 12 (D 64), 50 : 16 (128); 1 x 256 on 4000, 32 heads on 8, D 64 50 : 64; 12 heads on 2, D 128, 1 x 256 on
// 4000 58 : 58, 1 x 512 on 16000 118 : 276, 4 x 1024 on 4000 194 : 655.
bool fp8_prefill_tc_takes(int dtype, int head_dim, int64_t num_blocks, int block_size, int num_q_heads, int num_kv_heads,
                          int64_t num_seqs, int64_t max_seqlen_q, int64_t max_context, int sms) {
  if ((dtype != MI_DTYPE_BFLOAT16 && dtype != MI_DTYPE_FLOAT16) || (head_dim != 64 && head_dim != 128) || sms > kF8MaxCtas ||
      num_blocks >= (int64_t{1} << 31) / num_kv_heads / (block_size / kF8Group))  // places are 32 bits here
    return false;
  const int64_t rows = max_seqlen_q * (num_q_heads / num_kv_heads);
  const double tiles = static_cast<double>(num_seqs * num_kv_heads) * static_cast<double>((rows + 127) / 128) *
                       static_cast<double>((max_context + 127) / 128);
  return tiles * head_dim >= 640. * sms;
}

size_t fp8_prefill_tc_workspace(int head_dim, int sms) { return f8_prefill_workspace(head_dim, sms); }

// At most kF8MaxSeqs sequences.
cudaError_t launch_fp8_prefill_tc(const CodedPrefillParams &p, int dtype, int head_dim, cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16)
    return head_dim == 64 ? launch_tc<__nv_bfloat16, 64>(p, stream) : launch_tc<__nv_bfloat16, 128>(p, stream);
  return head_dim == 64 ? launch_tc<__half, 64>(p, stream) : launch_tc<__half, 128>(p, stream);
}

}  // namespace mi
