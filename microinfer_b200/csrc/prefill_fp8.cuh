// How the tcgen05 prefill over the 8-bit cache deals out its work, for the kernel, its join and what is done over behind it.
//
// A unit is 256 rows (token, query head of the group) of one sequence and kv head; it costs kUnitCost and, for each 128 keys that its
// last row sees, kPairCost, or kSingleCost where it has no more than 128 rows (a tile of one query tile takes
// about 4/7 of one of two; the start of a unit about as long as a tile).  Units in the order sequence, kv head,
// rows are one list of costs, cut into equal shares; a key tile belongs to the CTA in whose share it starts.
#pragma once

#include "common.cuh"
#include "fp8.cuh"
#include "params.cuh"

namespace mi {

constexpr int kF8MaxSeqs = 1024;  // of one launch (prefix sums in shared memory)
constexpr int kF8MaxCtas = 1024;
constexpr int kPairCost = 7, kSingleCost = 4, kUnitCost = 8;
constexpr int kLeastShare = 28;   // of a CTA: above kUnitCost + kPairCost, so every CTA inside a unit has a tile of it

struct F8Work {
  int64_t total, share;
};

// What a CTA leaves about the unit that goes on in the next one; parts 0: none.
struct F8Meta {
  int32_t seq, kvh, pair, parts;
};

// Workspace: [CTA][2][m, l, mean of V][256 rows], the part of a unit that began in an earlier CTA, then that of the one that
// goes on; the CTAs' F8Meta; a byte for each softmax warp that met what is to be done over (the first also for
// the warp that looks for NaN of V in groups of scale 0).
__host__ __device__ inline size_t f8_parts_bytes(int head_dim, int ctas) {
  return static_cast<size_t>(ctas) * 2 * 256 * (head_dim + 2) * sizeof(float);
}
__host__ __device__ inline size_t f8_prefill_workspace(int head_dim, int ctas) {
  return f8_parts_bytes(head_dim, ctas) + static_cast<size_t>(ctas) * (sizeof(F8Meta) + 8);
}
__device__ __forceinline__ F8Meta *f8_meta(const CodedPrefillParams &p, int head_dim, int ctas) {
  return reinterpret_cast<F8Meta *>(reinterpret_cast<uint8_t *>(p.workspace) + f8_parts_bytes(head_dim, ctas));
}
__device__ __forceinline__ uint8_t *f8_odd(const CodedPrefillParams &p, int head_dim, int ctas) {
  return reinterpret_cast<uint8_t *>(f8_meta(p, head_dim, ctas) + ctas);
}

// A sequence as its units see it.
struct F8Seq {
  int q0, rows, prefix, keys;  // rows of a kv head; positions before the chunk (negative: a context shorter than it); keys that exist
  __device__ __forceinline__ void load(const CodedPrefillParams &p, int64_t seq) {
    q0 = p.cu_seqlens_q[seq];
    const int64_t q_len = max(int64_t{0}, static_cast<int64_t>(p.cu_seqlens_q[seq + 1]) - q0);
    const int64_t ctx = static_cast<int64_t>(p.cu_seqlens_k[seq + 1]) - p.cu_seqlens_k[seq];
    // lengths that cannot be are work for the tokens that there are and one, which is flagged
    rows = static_cast<int>(min(min(q_len, p.num_tokens + 1) * (p.num_q_heads / p.num_kv_heads), int64_t{INT32_MAX} - 512));
    prefix = static_cast<int>(ctx - q_len);
    keys = static_cast<int>(max(int64_t{0}, min(ctx, p.bt_stride * p.block_size)));
  }
  __device__ __forceinline__ int pairs() const { return (rows + 255) / 256; }
  // 128-key tiles that rows up to `end` see
  __device__ __forceinline__ int tiles(const FastDiv &by_group, int end) const {
    const int seen = prefix + static_cast<int>(by_group.div(static_cast<uint32_t>(min(rows, end) - 1))) + 1;
    return (max(0, min(seen, keys)) + 127) / 128;
  }
  __device__ __forceinline__ int tile_cost(int pair) const { return rows - pair * 256 > 128 ? kPairCost : kSingleCost; }
  __device__ __forceinline__ int64_t cost(const FastDiv &by_group, int pair) const {
    return kUnitCost + static_cast<int64_t>(tiles(by_group, pair * 256 + 256)) * tile_cost(pair);
  }
};

// Prefix sums over the sequences' costs and the share of a CTA, by all threads of a block (a multiple of 32, at most 1024).
// prefix: [num_seqs + 1], scratch: [32], both shared.
__device__ __forceinline__ F8Work f8_work(const CodedPrefillParams &p, const FastDiv &by_group, int64_t *prefix, int64_t *scratch,
                                          int ctas) {
  const int n = static_cast<int>(p.num_seqs), threads = blockDim.x, per = (n + threads - 1) / threads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int i = 0; i < per; ++i) {
    const int s = threadIdx.x * per + i;
    if (s >= n) break;
    F8Seq q;
    q.load(p, s);
    int64_t cost = 0;
    for (int pair = 0; pair < q.pairs(); ++pair) cost += q.cost(by_group, pair);
    if (blockIdx.x == 0 && static_cast<int64_t>(p.cu_seqlens_k[s + 1]) - p.cu_seqlens_k[s] > p.bt_stride * p.block_size)
      flag_status(p.status, MI_DEV_BAD_BLOCK);
    prefix[s + 1] = cost;  // of one kv head, for now
    sum += cost * p.num_kv_heads;
  }
  int64_t incl = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int64_t before = incl - sum;
  for (int w = 0; w < warp; ++w) before += scratch[w];
  if (threadIdx.x == 0) prefix[0] = 0;
  for (int i = 0; i < per; ++i) {
    const int s = threadIdx.x * per + i;
    if (s >= n) break;
    before += prefix[s + 1] * p.num_kv_heads;
    prefix[s + 1] = before;
  }
  __syncthreads();
  F8Work w;
  w.total = prefix[n];
  w.share = max(int64_t{kLeastShare}, (w.total + ctas - 1) / ctas);
  return w;
}

// What a CTA does of a unit: key tiles j0 to j1 - 1, of query tile x those before end[x].
struct F8Item {
  int seq, q0, kvh, pair, row0, prefix, keys;
  int16_t rows[2];
  int end[2];
  int j0, j1;
  int parts;           // of a unit that goes on: CTAs that hold parts of it
  int16_t first, last;  // whether it has the unit's first tile, its last
};

// The items of a CTA, in order; every role walks them by itself.
struct F8Walker {
  int64_t lo, hi, at, share;  // this CTA's share, and the start of the next unit
  int seq, kvh, pair, n;
  F8Seq q;
  __device__ __forceinline__ void start(const CodedPrefillParams &p, const FastDiv &by_group, const int64_t *prefix,
                                        const F8Work &work, int cta) {
    share = work.share;
    lo = cta * share;
    hi = min(lo + share, work.total);
    n = static_cast<int>(p.num_seqs);
    seq = n, kvh = pair = 0, at = lo;
    if (lo >= hi) return;
    int a = 0, b = n - 1;  // the last sequence that does not start past `lo`
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (prefix[mid] <= lo)
        a = mid;
      else
        b = mid - 1;
    }
    seq = a;
    q.load(p, seq);
    const int64_t cost = (prefix[a + 1] - prefix[a]) / p.num_kv_heads;  // not 0: `lo` is in it
    kvh = static_cast<int>((lo - prefix[a]) / cost);
    at = prefix[a] + kvh * cost;
    for (;;) {
      const int64_t c = q.cost(by_group, pair);
      if (at + c > lo) break;
      at += c;
      ++pair;
    }
  }
  __device__ __forceinline__ bool next(const CodedPrefillParams &p, const FastDiv &by_group, F8Item &it) {
    while (at < hi && seq < n) {
      const int ct = q.tile_cost(pair), tiles = q.tiles(by_group, pair * 256 + 256);
      const int64_t c0 = at, begin = at + kUnitCost;  // tile j > 0 starts at begin + j * ct, tile 0 with the unit
      it.seq = seq, it.q0 = q.q0, it.kvh = kvh, it.pair = pair, it.row0 = pair * 256, it.prefix = q.prefix, it.keys = q.keys;
      it.rows[0] = static_cast<int16_t>(min(128, q.rows - it.row0));
      it.rows[1] = static_cast<int16_t>(max(0, min(128, q.rows - it.row0 - 128)));
      it.j0 = lo > c0 ? max(1, static_cast<int>((lo - begin + ct - 1) / ct)) : 0;
      it.j1 = hi < begin + static_cast<int64_t>(tiles) * ct ? min(tiles, max(1, static_cast<int>((hi - begin + ct - 1) / ct)))
                                                            : tiles;
      it.first = it.j0 == 0, it.last = it.j1 == tiles;
      it.end[0] = min(it.j1, q.tiles(by_group, it.row0 + 128));
      it.end[1] = it.rows[1] > 0 ? it.j1 : it.j0;
      it.parts = static_cast<int>((begin + static_cast<int64_t>(tiles - 1) * ct) / share - c0 / share) + 1;
      at = begin + static_cast<int64_t>(tiles) * ct;
      if (++pair == q.pairs()) {
        pair = 0;
        if (++kvh == p.num_kv_heads) {
          kvh = 0;
          while (++seq < n) {
            q.load(p, seq);
            if (q.rows > 0) break;
          }
        }
      }
      if (it.j0 < it.j1 || (tiles == 0 && it.j0 == 0)) return true;
    }
    return false;
  }
};

}  // namespace mi
