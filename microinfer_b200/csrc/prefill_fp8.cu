// Causal chunked prefill straight from the 8-bit cache (layout: fp8.cuh) on the warp-level tensor cores, for what the tcgen05
// kernels do not take (fp32, head_dims other than 64 and 128), for little work, and for what they leave to be done over.
//
// A CTA takes 128 rows of one kv head, a row being (token, query head of the group), so any group
// fills the tiles; 8 warps of 16 rows.  It walks the keys 64 at a time: the codes of the next tile are on their
// way into shared memory (16-byte cp.async) while this one is worked on, then become f16 rows in the other half, decoded
// once for the 8 warps by one conversion for two codes.  The scales stay out of them: a group of 16 keys has one for K, which
// goes into the factor that its scores meet on their way into the exponential, and one for V, which goes into the exponent of
// its p.  So f16 is exact for every type of query, and an element costs what it would without scales.
// S = Q K^T and O += P V are m16n8k16 with fp32 accumulators, P passes from the one to the other in registers; online
// softmax in fp32, the maximum followed 3 binades behind at most.  q rows are multiplied by a power of two that puts their
// largest element into [2^14, 2^15); fp32 goes in as two f16 parts (22 bits), as does its p.
// V's scale: O is held in units of 2^(R - 127), R a running reference at or above every group's byte, and p goes in as
// p * 2^(byte - R) * 2^12, which keeps a key 2^-19 of the largest at full precision 7 binades below R.  Tiles with a group
// further below (or a zero one) take their groups one by one and add them in fp32; a group above raises R.
// NaN of V are held as zeros and set in the rows that see the key, so they never reach rows before it.
// Few rows over a long context are split over the keys; a second launch joins the splits, as means of V.
//
// Measured (cold L2): 1 x 64 rows on 64 keys 12 us (head_dim 64) and 16 us (128), 16 x 64 on 64 the same, 1 x 512 on 512 30 to 34.
// Larger calls it does at 170 to 190 TFLOP/s of head_dim 64, half of what the tcgen05 kernel does: the exponentials and the decoding
// share the issue slots of the warps that also feed the MMAs.
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.cuh"
#include "params.cuh"
#include "prefill_fp8.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kRows = 128;
constexpr int kThreads = 256;
constexpr int kFactorMax = 94;  // largest exponent of a score's factor: sums of products are below 2^32
constexpr int kNear = 7;        // binades below R that p takes in
constexpr float kLift = 12.f, kLag = 3.f;  // p <= 2^(kLift + kLag) is within f16
constexpr float kExact = 0x1p20f;          // m up to here is off by 2^-4 at most

// NB blocks of 32 dims.
template <typename T, int NB>
struct P8Cfg {
  static constexpr bool kSplit = std::is_same<T, float>::value;
  static constexpr int kParts = kSplit ? 2 : 1;  // f16 parts of q and p
  static constexpr int D = NB * 32;
  static constexpr int kKeys = kSplit && NB > 4 ? 32 : 64;  // of a tile: both parts of q leave room for so many
  static constexpr int kGroups = kKeys / kF8Group;
  static constexpr int kRowBytes = (NB + 1) / 2 * 128;  // f16 rows of whole 128 bytes, for the swizzle
  static constexpr int kTile = kKeys * kRowBytes;       // K or V of a tile
  static constexpr int kQuery = kRows * kRowBytes;      // one part of q
  static constexpr int kChunks = 2 * kGroups * D;       // 16-byte chunks of codes of a tile, K and V
  static constexpr int kPer = (kChunks + kThreads - 1) / kThreads;  // of those per thread
  static constexpr int kRaw = kPer * kThreads * 16;     // codes on their way
  static constexpr int kMisc = kRows * 4 + 2 * (2 * kGroups * 4 + kGroups * 8 + kKeys);
  static constexpr int kSmem = kParts * kQuery + 4 * kTile + kRaw + kMisc;
  static constexpr int kCtas = kSmem <= 113 * 1024 ? 2 : 1;  // of an SM
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// Byte offset of 16-byte chunk c of a row, chunks swizzled so that 8 rows' accesses to one chunk touch every bank.
template <int NB>
__device__ __forceinline__ uint32_t at(int row, int c) {
  return static_cast<uint32_t>(row * ((NB + 1) / 2 * 128) + ((c ^ (row & 7)) << 4));
}

__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// What a value leaves after its rounding to f16.
__device__ __forceinline__ float rest16(float x) { return x - __half2float(__float2half_rn(x)); }
// 2^e for any e, through two factors where one has no normal exponent.
__device__ __forceinline__ float exp2i(int e) {
  const int a = max(-126, min(127, e)), b = max(-126, min(127, e - a));
  return __uint_as_float(static_cast<uint32_t>(a + 127) << 23) * __uint_as_float(static_cast<uint32_t>(b + 127) << 23);
}

// Place of V's code of a token and dim in a group.
__device__ __forceinline__ int value_place(int tok, int dim, int head_dim) {
  const F8Place r = f8_place(dim >> 3, head_dim);
  return r.v + (dim & 4 ? r.split : 0) + (dim & 3) * 2 + (tok >> 3) * r.half + ((tok & 7) >> 1) * r.pair + (tok & 1);
}

}  // namespace

// 128 rows of one kv head against the keys of one split.
template <typename T, int NB>
__device__ __forceinline__ void prefill_tile(const CodedPrefillParams &p, const FastDiv &by_group, const FastDiv &by_page,
                                             int seq, int kvh, int tile, int split) {
  using C = P8Cfg<T, NB>;
  constexpr int D = C::D, kParts = C::kParts, kKeys = C::kKeys, kGroups = C::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *tiles = smem + kParts * C::kQuery;  // [2][K, V]
  uint8_t *raw = tiles + 4 * C::kTile;         // codes of the next tile, each thread's its own
  int *row_exp = reinterpret_cast<int *>(raw + C::kRaw);  // [rows]: exponent that a row's products want, without K's scale
  int *bytes = row_exp + kRows;                // [2][K, V][groups]: scale bytes, -1 where the page is none (V's past the keys too)
  int64_t *where = reinterpret_cast<int64_t *>(bytes + 4 * kGroups);  // [2][groups]: places in the pools, -1 past the keys, -2: the page is none
  uint8_t *marks = reinterpret_cast<uint8_t *>(where + 2 * kGroups);  // [2][keys]: blocks of 32 dims of V with a NaN, a bit each
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int64_t q0 = p.cu_seqlens_q[seq];
  const int64_t q_len = p.cu_seqlens_q[seq + 1] - q0;
  const int64_t row0 = static_cast<int64_t>(tile) * kRows;
  if (row0 >= q_len * G) return;
  int64_t ctx = static_cast<int64_t>(p.cu_seqlens_k[seq + 1]) - p.cu_seqlens_k[seq];
  const int64_t prefix = ctx - q_len;
  if (ctx > p.bt_stride * p.block_size) {
    if (threadIdx.x == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    ctx = p.bt_stride * p.block_size;
  }
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), q_len * G - row0));
  const int64_t last_pos = prefix + by_group.div(static_cast<uint32_t>(row0 + rows - 1));
  const int keys = static_cast<int>(max(int64_t{0}, min(ctx, last_pos + 1)));
  const int all_tiles = (keys + kKeys - 1) / kKeys;
  const int per_split = (all_tiles + p.num_splits - 1) / p.num_splits;
  const int k_begin = split * per_split, k_end = min(all_tiles, k_begin + per_split);

  const F8Scale scale = f8_softmax_scale(p.scale_log2);  // its exponent goes to the rows'
  const float mantissa = scale.mantissa;

  // ---- copies of a tile's codes: a thread's chunks, in the order of memory, K's, then V's ----
  struct Chunk {
    bool exists, value;
    int group, i;  // chunk i of the group
  };
  auto chunk = [&](int n) {
    const int id = n * kThreads + static_cast<int>(threadIdx.x);
    Chunk c;
    c.exists = C::kChunks % kThreads == 0 || id < C::kChunks;
    c.value = id >= C::kChunks / 2;
    const int in = c.value ? id - C::kChunks / 2 : id;
    c.group = in / D, c.i = in % D;
    return c;
  };
  const int per_page = p.block_size / kF8Group;
  const int32_t *table = p.block_tables + seq * p.bt_stride;
  // Group `index` of the context: its place in the pools from the page that the table names.
  auto page_of = [&](uint32_t index) {
    return static_cast<int64_t>(index) * kF8Group < keys ? __ldg(table + by_page.div(index)) : INT32_MIN;
  };
  auto place_of = [&](uint32_t index, int page) -> int64_t {
    if (page == INT32_MIN && static_cast<int64_t>(index) * kF8Group >= keys) return -1;
    if (page < 0 || page >= p.num_blocks) return -2;
    return (static_cast<int64_t>(page) * p.num_kv_heads + kvh) * per_page + (index - by_page.div(index) * per_page);
  };
  // The pages of a tile's groups are looked up by a thread each, two tiles ahead of the products and one of the copies.
  int my_page = INT32_MIN;
  auto look_up = [&](int kt) {
    if (threadIdx.x < kGroups) my_page = page_of(static_cast<uint32_t>(kt) * kGroups + threadIdx.x);
  };
  auto looked_up = [&](int kt) {
    if (threadIdx.x < kGroups)
      where[(kt & 1) * kGroups + threadIdx.x] = place_of(static_cast<uint32_t>(kt) * kGroups + threadIdx.x, my_page);
  };
  const uint32_t my_raw = smem_addr(raw) + threadIdx.x * 16;
  int my_scale = 0;  // of the first threads, a group each of K, then of V
  auto fetch = [&](int kt) {
#pragma unroll
    for (int n = 0; n < C::kPer; ++n) {
      const Chunk c = chunk(n);
      const int64_t place = c.exists ? where[(kt & 1) * kGroups + c.group] : -1;
      const uint8_t *from = (c.value ? p.value_pages : p.key_pages) + max(place, int64_t{0}) * f8_group_bytes(D) + c.i * 16;
      const int size = place < 0 ? 0 : 16;  // keys that do not exist: zeros
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(my_raw + n * kThreads * 16), "l"(from), "r"(size)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (threadIdx.x < 2 * kGroups) {
      const int64_t place = where[(kt & 1) * kGroups + threadIdx.x % kGroups];
      const uint8_t *pool = threadIdx.x < kGroups ? p.key_pages : p.value_pages;
      my_scale = place < 0 ? (place == -2 || threadIdx.x >= kGroups ? -1 : 0) : pool[place * f8_group_bytes(D) + kF8Group * D];
    }
  };
  // This thread's chunks as f16 rows of buffer `buf`; whether V has a NaN among them.
  auto place = [&](int buf) -> bool {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    bool nan = false;
#pragma unroll
    for (int n = 0; n < C::kPer; ++n) {
      const Chunk c = chunk(n);
      if (!c.exists) continue;
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(my_raw + n * kThreads * 16));
      uint8_t *to = tiles + (buf * 2 + c.value) * C::kTile;
      const int part = c.i / 64, i = c.i % 64, first = c.group * kF8Group;
      const bool full = NB % 2 == 0 || part < NB / 2;
      if (c.value) {
        if (f8_any_nan(w[0]) || f8_any_nan(w[1]) || f8_any_nan(w[2]) || f8_any_nan(w[3])) {
          nan = true;
#pragma unroll
          for (int u = 0; u < 4; ++u) {  // 0x7f and 0xff to zero
            const uint32_t is = ((w[u] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            w[u] &= ~(is | (is - (is >> 7)));
          }
        }
        uint32_t h[8];  // pairs of tokens, dim after dim
#pragma unroll
        for (int u = 0; u < 4; ++u) f8_to_f16(w[u], h[2 * u], h[2 * u + 1]);
        if (full) {  // 8 dims of a pair
          const int tok = first + i / 32 * 8 + i % 4 * 2, at_chunk = part * 8 + i % 32 / 4;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = __byte_perm(h[2 * u], h[2 * u + 1], k ? 0x7632 : 0x5410);
            *reinterpret_cast<uint4 *>(to + at<NB>(tok + k, at_chunk)) = make_uint4(r[0], r[1], r[2], r[3]);
          }
        } else {  // 4 dims of two pairs
          const int tok = first + i / 16 * 8 + i % 2 * 4, dims4 = i % 16 / 2;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t *s = h + k / 2 * 4;
            const uint32_t r0 = __byte_perm(s[0], s[1], k & 1 ? 0x7632 : 0x5410);
            const uint32_t r1 = __byte_perm(s[2], s[3], k & 1 ? 0x7632 : 0x5410);
            *reinterpret_cast<uint2 *>(to + at<NB>(tok + k, part * 8 + dims4 / 2) + dims4 % 2 * 8) = make_uint2(r0, r1);
          }
        }
      } else {
        uint32_t h[8];
#pragma unroll
        for (int u = 0; u < 4; ++u) f8_to_f16(w[u], h[2 * u], h[2 * u + 1]);
        const int tok = first + (full ? i / 4 : i / 2), c16 = part * 8 + (full ? i % 4 : i % 2) * 2;
        *reinterpret_cast<uint4 *>(to + at<NB>(tok, c16)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(to + at<NB>(tok, c16 + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    }
    if (threadIdx.x < 2 * kGroups) {
      bytes[buf * 2 * kGroups + threadIdx.x] = my_scale;
      if (my_scale < 0 && threadIdx.x < kGroups) flag_status(p.status, MI_DEV_BAD_BLOCK);
    }
    if (threadIdx.x < kKeys) marks[buf * kKeys + threadIdx.x] = 0;
    return nan;
  };
  // Marks of this thread's NaN of V, whose codes are still in `raw`.
  auto mark = [&](int buf, int kt) {
    for (int n = 0; n < C::kPer; ++n) {
      const Chunk c = chunk(n);
      if (!c.exists || !c.value) continue;
      const int part = c.i / 64, i = c.i % 64;
      const bool full = NB % 2 == 0 || part < NB / 2;
      for (int b = 0; b < 16; ++b) {
        if ((raw[(n * kThreads + threadIdx.x) * 16 + b] & 0x7f) != 0x7f) continue;
        const int tok = full ? i / 32 * 8 + i % 4 * 2 + (b & 1) : i / 16 * 8 + i % 2 * 4 + b / 8 * 2 + (b & 1);
        const int dim = part * 64 + (full ? i % 32 / 4 * 8 + b / 2 : i % 16 / 2 * 4 + b % 8 / 2);
        const int key = c.group * kF8Group + tok;
        if (kt * kKeys + key < keys)
          atomicOr(reinterpret_cast<unsigned *>(marks + buf * kKeys) + key / 4, 1u << (key % 4 * 8 + dim / 32));
      }
    }
  };
  auto arrive = [&](int buf, int kt) -> bool {
    looked_up(kt + 1);
    const bool mine = place(buf);
    const bool any = __syncthreads_or(mine);
    if (any) {
      if (mine) mark(buf, kt);
      __syncthreads();
    }
    return any;
  };

  if (k_begin < k_end) {
    look_up(k_begin);
    looked_up(k_begin);
    look_up(k_begin + 1);
    __syncthreads();
    fetch(k_begin);
  }

  // ---- q into shared memory, as `kParts` operands: four lanes to a row, 8 of every 32 dims each ----
#pragma unroll 1
  for (int r = threadIdx.x / 4; r < kRows; r += kThreads / 4) {
    const uint32_t row = static_cast<uint32_t>(row0) + r;
    const int64_t token = q0 + by_group.div(row);
    const bool there = r < rows && token >= 0 && token < p.num_tokens;
    const T *src = static_cast<const T *>(p.query) +
                   (there ? (token * p.num_q_heads + kvh * G + (row - by_group.div(row) * G)) * D : 0);
    float x[NB][8];
    uint32_t top = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[b][u] = 0.f;
      if (there) {
        if constexpr (C::kSplit) {
          const float4 *f = reinterpret_cast<const float4 *>(src + b * 32 + t * 8);
          const float4 lo = f[0], hi = f[1];
          x[b][0] = lo.x, x[b][1] = lo.y, x[b][2] = lo.z, x[b][3] = lo.w;
          x[b][4] = hi.x, x[b][5] = hi.y, x[b][6] = hi.z, x[b][7] = hi.w;
        } else {
          float2 f[4];
          Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(src + b * 32 + t * 8), f);
#pragma unroll
          for (int u = 0; u < 4; ++u) x[b][2 * u] = f[u].x, x[b][2 * u + 1] = f[u].y;
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) top = max(top, __float_as_uint(x[b][u]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(kAll, top, 1));
    top = max(top, __shfl_xor_sync(kAll, top, 2));
    // not finite: as it is; nor do zeros need a power
    const int e = top >= 0x7f800000u || top == 0 || scale.sign == 0.f ? 0 : min(14 - (static_cast<int>(top >> 23) - 127), 126);
    const float f = exp2i(e) * scale.sign;
    if (t == 0) row_exp[r] = scale.exponent - e;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[b][u] *= f;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        *reinterpret_cast<uint4 *>(smem + part * C::kQuery + at<NB>(r, b * 4 + t)) =
            make_uint4(pack16(x[b][0], x[b][1]), pack16(x[b][2], x[b][3]), pack16(x[b][4], x[b][5]), pack16(x[b][6], x[b][7]));
        if (part + 1 < kParts)
#pragma unroll
          for (int u = 0; u < 8; ++u) x[b][u] = rest16(x[b][u]);
      }
    }
  }

  bool has_nan = false;
  if (k_begin < k_end)
    has_nan = arrive(0, k_begin);
  else
    __syncthreads();

  // this thread's rows: g and g + 8 of its warp's 16
  int pos[2], rexp[2];  // positions are below 2^31 as contexts are
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = warp * 16 + g + 8 * i;
    pos[i] = r < rows ? static_cast<int>(prefix + by_group.div(static_cast<uint32_t>(row0) + r)) : -1;
    rexp[i] = row_exp[r];
  }
  const int first_pos = static_cast<int>(prefix + by_group.div(static_cast<uint32_t>(row0) + min(warp * 16, rows - 1)));
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  int ref = -1;  // R; the same in every thread

  // ldmatrix addresses: the swizzle only touches bits 4 to 6, so a lane's row and chunk parity go into a
  // base and even chunk 2n is one exclusive or (and an immediate offset past 8 chunks)
  const int mi = lane >> 3, rr = lane & 7;
  const uint32_t q_lane = (smem_addr(smem) + (warp * 16 + (mi & 1) * 8 + rr) * C::kRowBytes) | ((rr ^ (mi >> 1)) << 4);
  const uint32_t k_lane = (((mi >> 1) * 8 + rr) * C::kRowBytes) | ((rr ^ (mi & 1)) << 4);
  const uint32_t v_lane = (((mi & 1) * 8 + rr) * C::kRowBytes) | ((rr ^ (mi >> 1)) << 4);
  const uint32_t t_base = smem_addr(tiles);
  auto even_chunk = [](uint32_t lane_base, int n) { return (lane_base ^ ((2 * n & 7) << 4)) + (n >> 2) * 128; };
#pragma unroll 1
  for (int kt = k_begin; kt < k_end; ++kt) {
    const int buf = (kt - k_begin) & 1;
    const bool more = kt + 1 < k_end;
    if (more) {
      fetch(kt + 1);
      look_up(kt + 2);
    }
    const uint32_t k_base = t_base + buf * 2 * C::kTile + k_lane;
    const uint32_t v_base = t_base + buf * 2 * C::kTile + C::kTile + v_lane;
    float s[kKeys / 8][4];
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t a[kParts][4];
#pragma unroll
      for (int part = 0; part < kParts; ++part) ldsm(even_chunk(q_lane, ks) + part * C::kQuery, a[part]);
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {  // 16 keys: dims lo, hi of keys 0-7, then of keys 8-15
        uint32_t b[4];
        ldsm(even_chunk(k_base, ks) + n * 16 * C::kRowBytes, b);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          mma(s[2 * n], a[part], b[0], b[1]);
          mma(s[2 * n + 1], a[part], b[2], b[3]);
        }
      }
    }
    // the groups' scales: K's into the factors of their scores, V's against R
    const int key0 = kt * kKeys;
    int kb[kGroups], vb[kGroups];
    bool pages = true, far_scores = false;
    int v_top = -1, v_low = 255;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      kb[i] = bytes[buf * 2 * kGroups + i], vb[i] = bytes[buf * 2 * kGroups + kGroups + i];
      pages &= kb[i] >= 0;
      far_scores |= kb[i] - 127 + max(rexp[0], rexp[1]) > kFactorMax;
      v_top = max(v_top, vb[i]);
      if (vb[i] >= 0) v_low = min(v_low, vb[i]);
    }
    if (v_top > ref) {  // uniform in the CTA
      const int next = v_top + 2;  // two binades of room
      if (ref >= 0) {
        const float f = exp2i(ref - next);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] *= f, o[n][1] *= f, o[n][2] *= f, o[n][3] *= f;
      }
      ref = next;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) vb[i] = vb[i] < 0 ? ref : vb[i];  // its keys have no p
    const bool far_values = v_low == 0 || ref - v_low > kNear;  // uniform in the CTA; a byte of 0 is no exponent
    float factor[kGroups][2];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = kb[i] == 0 ? -126 : max(-126, min(kFactorMax, kb[i] - 127 + rexp[u]));  // further down every score is 0
        factor[i][u] = __uint_as_float(static_cast<uint32_t>(e + 127) << 23) * mantissa;
      }
    if (__any_sync(kAll, far_scores)) {
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int e = kb[i / 2] == 0 ? 0 : kb[i / 2] - 127 + rexp[u >> 1] - kFactorMax;
          if (e > 0) s[i][u] *= exp2i(e);
        }
    }
    if (key0 + kKeys - 1 > first_pos || key0 + kKeys > keys || !pages) {  // uniform in the warp
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
        const int key = key0 + i * 8 + 2 * t;
        const bool none = kb[i / 2] < 0;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (key + (u & 1) > min(pos[u >> 1], keys - 1) || none) s[i][u] = -INFINITY;
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        top[u] = fmaxf(top[u], fmaxf(fmaxf(s[2 * i][2 * u], s[2 * i][2 * u + 1]),
                                     fmaxf(s[2 * i + 1][2 * u], s[2 * i + 1][2 * u + 1])) * factor[i][u]);
    if (__any_sync(kAll, top[0] - m[0] > kLag || top[1] - m[1] > kLag)) {  // m + kLag may round to m + 4 from 2^24 on
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(kAll, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(kAll, top[i], 2));
        const float next = fmaxf(m[i], top[i]);
        const float f = m[i] == -INFINITY ? 0.f : fast_exp2(m[i] - next);
        l[i] *= f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][2 * i] *= f, o[n][2 * i + 1] *= f;
        m[i] = next;
      }
    }
    float high[2] = {m[0], m[1]};
    if (__any_sync(kAll, fmaxf(fabsf(m[0] == -INFINITY ? 0.f : m[0]), fabsf(m[1] == -INFINITY ? 0.f : m[1])) > kExact)) {
      // m rounds away more than a product less it may be off by: the product rounds as m did, and m goes at once
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u)  // a row without an m has masked scores and NaN, which stay
          s[i][u] = __fmul_rn(s[i][u], factor[i / 2][u >> 1]) - (m[u >> 1] == -INFINITY ? 0.f : m[u >> 1]);
#pragma unroll
      for (int i = 0; i < kGroups; ++i) factor[i][0] = factor[i][1] = 1.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) high[u] = m[u] == -INFINITY ? m[u] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int below = far_values ? 0 : vb[i] - ref;  // p goes in times 2^below
      const float back = __uint_as_float(static_cast<uint32_t>(127 - below) << 23);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float base = high[u] == -INFINITY ? 0.f : kLift - high[u] + static_cast<float>(below);  // no key yet: exp2(-inf) = 0
        float sum = 0.f;
#pragma unroll
        for (int n = 2 * i; n < 2 * i + 2; ++n)
#pragma unroll
          for (int v = 2 * u; v < 2 * u + 2; ++v) {
            s[n][v] = fast_exp2(fmaf(s[n][v], factor[i][u], base));
            sum += s[n][v];
          }
        l[u] = fmaf(sum, back, l[u]);
      }
    }
    auto operands = [&](int ks, uint32_t (&a)[kParts][4]) {
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          a[part][2 * u] = pack16(s[2 * ks + u][0], s[2 * ks + u][1]);
          a[part][2 * u + 1] = pack16(s[2 * ks + u][2], s[2 * ks + u][3]);
          if (part + 1 < kParts)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[2 * ks + u][c] = rest16(s[2 * ks + u][c]);
        }
      }
    };
    if (!far_values) {
#pragma unroll
      for (int ks = 0; ks < kGroups; ++ks) {
        uint32_t a[kParts][4];
        operands(ks, a);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {  // 16 dims: keys lo, hi of dims 0-7, then of dims 8-15
          uint32_t b[4];
          ldsm_t(even_chunk(v_base, n) + ks * 16 * C::kRowBytes, b);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            mma(o[2 * n], a[part], b[0], b[1]);
            mma(o[2 * n + 1], a[part], b[2], b[3]);
          }
        }
      }
    } else {  // group by group
#pragma unroll
      for (int ks = 0; ks < kGroups; ++ks) {
        uint32_t a[kParts][4];
        operands(ks, a);
        const float back = vb[ks] == 0 ? 0.f : exp2i(vb[ks] - ref);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          ldsm_t(even_chunk(v_base, n) + ks * 16 * C::kRowBytes, b);
          float r[2][4] = {};
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            mma(r[0], a[part], b[0], b[1]);
            mma(r[1], a[part], b[2], b[3]);
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) o[2 * n + u / 4][u % 4] = fmaf(r[u / 4][u % 4], back, o[2 * n + u / 4][u % 4]);
        }
      }
    }
    if (has_nan) {  // uniform in the CTA
#pragma unroll 1
      for (int key = 0; key < kKeys; ++key) {
        const unsigned blocks = marks[buf * kKeys + key];
        if (!blocks) continue;
        const uint32_t index = static_cast<uint32_t>(kt) * kGroups + key / kF8Group;
        const uint8_t *codes = p.value_pages + place_of(index, page_of(index)) * f8_group_bytes(D);  // it has a page
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          if (!(blocks >> (n / 4) & 1u)) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (key0 + key <= pos[u >> 1] && (codes[value_place(key % kF8Group, n * 8 + 2 * t + (u & 1), D)] & 0x7f) == 0x7f)
              o[n][u] = __uint_as_float(0x7fffffffu);
        }
      }
    }
    if (more) has_nan = arrive(buf ^ 1, kt + 1);
  }

  const float unit = exp2i(ref - 127);  // no keys: o is 0
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(kAll, l[i], 1);
    l[i] += __shfl_xor_sync(kAll, l[i], 2);
    const int r = warp * 16 + g + 8 * i;
    if (r >= rows) continue;
    const uint32_t row = static_cast<uint32_t>(row0) + r;
    const int64_t token = q0 + by_group.div(row);
    if (token < 0 || token >= p.num_tokens) {
      flag_status(p.status, MI_DEV_BAD_SLOT);
      continue;
    }
    const int64_t at_row = token * p.num_q_heads + kvh * G + (row - by_group.div(row) * G);
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    if (p.num_splits == 1) {
      T *out = static_cast<T *>(p.out) + at_row * D + 2 * t;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const float a = o[n][2 * i] * inv * unit, b = o[n][2 * i + 1] * inv * unit;
        if constexpr (C::kSplit) {
          *reinterpret_cast<float2 *>(out + n * 8) = make_float2(a, b);
        } else {
          const T pair[2] = {Elem<T>::from_float(a), Elem<T>::from_float(b)};
          *reinterpret_cast<uint32_t *>(out + n * 8) = *reinterpret_cast<const uint32_t *>(pair);
        }
      }
    } else {
      float *st = p.workspace + (split * p.num_tokens * p.num_q_heads + at_row) * (D + 2);
      if (t == 0) st[0] = m[i], st[1] = l[i];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2 *>(st + 2 + n * 8 + 2 * t) = make_float2(o[n][2 * i] * inv * unit, o[n][2 * i + 1] * inv * unit);
    }
  }
}

template <typename T, int NB>
__global__ void __launch_bounds__(kThreads, P8Cfg<T, NB>::kCtas)
    fp8_prefill_kernel(const CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page) {
  pdl_wait();
  const unsigned at = gridDim.x - 1 - blockIdx.x;  // the last rows, with the most keys, first
  prefill_tile<T, NB>(p, by_group, by_page, blockIdx.z, blockIdx.y, at / p.num_splits, at % p.num_splits);
  pdl_launch_dependents();
}

// After the dense kernel: the sequences and kv heads of which the gather has noted that it cannot do them, over again.  Hardly
// ever any, so a few CTAs look and take all tiles if so.
template <typename T, int NB>
__global__ void __launch_bounds__(kThreads, P8Cfg<T, NB>::kCtas)
    fp8_prefill_redo_gathered_kernel(const CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page, int tiles) {
  pdl_wait();
  const int64_t ctx = static_cast<int64_t>(p.cu_seqlens_k[blockIdx.z + 1]) - p.cu_seqlens_k[blockIdx.z];
  const int64_t groups = min((ctx + kF8Group - 1) / kF8Group, static_cast<int64_t>(p.redo_groups));
  const uint8_t *noted = p.redo + (static_cast<int64_t>(blockIdx.z) * p.num_kv_heads + blockIdx.y) * p.redo_stride;
  bool any = false;
  for (int64_t i = threadIdx.x; i < groups; i += kThreads) any |= noted[i] != 0;
  if (__syncthreads_or(any))
    for (int tile = tiles - 1 - blockIdx.x; tile >= 0; tile -= gridDim.x) {
      prefill_tile<T, NB>(p, by_group, by_page, blockIdx.z, blockIdx.y, tile, 0);
      __syncthreads();  // every warp has read what the next tile overwrites
    }
  pdl_launch_dependents();
}

// After the tcgen05 kernel: the sequences and kv heads in whose CTAs it met what it cannot do, over again.  Hardly ever any.
// Their tiles are dealt out in turn, across them: short chunks have one each.
template <typename T, int NB>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_prefill_redo_kernel(const CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page, int ctas) {
  __shared__ int64_t prefix[kF8MaxSeqs + 1], scratch[32];
  __shared__ bool met[kF8MaxCtas];
  pdl_wait();
  const uint64_t *odd = reinterpret_cast<const uint64_t *>(f8_odd(p, NB * 32, ctas));  // a byte for each warp of a CTA
  bool any = false;
  for (int i = threadIdx.x; i < ctas; i += kThreads) any |= met[i] = odd[i] != 0;
  if (!__syncthreads_or(any)) {
    pdl_launch_dependents();
    return;
  }
  const F8Work work = f8_work(p, by_group, prefix, scratch, ctas);
  const int grid = gridDim.x;
  int turn = blockIdx.x;  // tiles until this CTA's next
  for (int seq = 0; seq < p.num_seqs; ++seq) {
    const int64_t cost = (prefix[seq + 1] - prefix[seq]) / p.num_kv_heads;
    if (cost == 0) continue;
    F8Seq q;
    q.load(p, seq);
    for (int kvh = 0; kvh < p.num_kv_heads; ++kvh) {
      const int64_t from = prefix[seq] + kvh * cost;
      const int first = static_cast<int>(from / work.share), last = static_cast<int>((from + cost - 1) / work.share);
      any = false;
      for (int i = first; i <= last; ++i) any |= met[i];
      if (!any) continue;
      const int tiles = (q.rows + kRows - 1) / kRows;
      for (; turn < tiles; turn += grid) {
        prefill_tile<T, NB>(p, by_group, by_page, seq, kvh, turn, 0);
        __syncthreads();  // every warp has read what the next tile overwrites
      }
      turn -= tiles;
    }
  }
  pdl_launch_dependents();
}

// Join the splits: a warp to a row, the rows of the sequences only.  A split's part is a mean of V, its m and its l.
template <typename T, int NB>
__global__ void __launch_bounds__(kThreads) fp8_prefill_join_kernel(const CodedPrefillParams p, const FastDiv by_group) {
  constexpr int D = NB * 32;
  pdl_wait();
  const int seq = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 31;
  const int G = p.num_q_heads / p.num_kv_heads;
  const int64_t q0 = p.cu_seqlens_q[seq];
  const int64_t rows = (p.cu_seqlens_q[seq + 1] - q0) * G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (row < rows) {
    const int64_t token = q0 + by_group.div(static_cast<uint32_t>(row));
    if (token >= 0 && token < p.num_tokens) {
      const int64_t at_row =
          token * p.num_q_heads + kvh * G + (row - by_group.div(static_cast<uint32_t>(row)) * static_cast<int64_t>(G));
      const int64_t stride = p.num_tokens * p.num_q_heads * (D + 2);
      const float *st = p.workspace + at_row * (D + 2);
      float M = -INFINITY, L = 0.f, A[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) A[b] = 0.f;
#pragma unroll 4
      for (int s = 0; s < p.num_splits; ++s, st += stride) {
        const float m = __ldcg(st), l = __ldcg(st + 1);
        float a[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) a[b] = __ldcg(st + 2 + b * 32 + lane);
        if (m == -INFINITY && l == 0.f) continue;  // no keys
        const float next = fmaxf(M, m);
        const float f = M == -INFINITY ? (L == 0.f ? 0.f : 1.f) : fast_exp2(M - next);
        const float e = m == -INFINITY ? 1.f : fast_exp2(m - next);
        const float sum = f * L + e * l, share = sum == 0.f ? 0.f : e * l / sum;  // of this part in the mean
#pragma unroll
        for (int b = 0; b < NB; ++b) A[b] = fmaf(share, a[b], A[b] - share * A[b]);
        L = sum;
        M = next;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
        static_cast<T *>(p.out)[at_row * D + b * 32 + lane] = Elem<T>::from_float(A[b]);
    }
  }
  pdl_launch_dependents();
}

namespace {

template <typename T, int NB>
cudaError_t launch_p8(const CodedPrefillParams &p, int64_t num_seqs, int64_t max_seqlen_q, cudaStream_t stream) {
  using C = P8Cfg<T, NB>;
  auto kern = fp8_prefill_kernel<T, NB>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int G = p.num_q_heads / p.num_kv_heads;
  const int64_t tiles = (max_seqlen_q * G + kRows - 1) / kRows;
  const FastDiv by_group(G), by_page(p.block_size / kF8Group);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(tiles * p.num_splits), p.num_kv_heads,
                                        static_cast<unsigned>(num_seqs)),
                             dim3(kThreads), C::kSmem, stream, p, by_group, by_page);
  if (e == cudaSuccess && p.num_splits > 1)
    e = launch_pdl(fp8_prefill_join_kernel<T, NB>,
                   dim3(static_cast<unsigned>((max_seqlen_q * G + kThreads / 32 - 1) / (kThreads / 32)),
                        p.num_kv_heads, static_cast<unsigned>(num_seqs)),
                   dim3(kThreads), 0, stream, p, by_group);
  return e;
}

template <typename T>
cudaError_t launch_p8_t(const CodedPrefillParams &p, int head_dim, int64_t num_seqs, int64_t max_seqlen_q,
                        cudaStream_t stream) {
  switch (head_dim / 32) {
    case 1: return launch_p8<T, 1>(p, num_seqs, max_seqlen_q, stream);
    case 2: return launch_p8<T, 2>(p, num_seqs, max_seqlen_q, stream);
    case 3: return launch_p8<T, 3>(p, num_seqs, max_seqlen_q, stream);
    case 4: return launch_p8<T, 4>(p, num_seqs, max_seqlen_q, stream);
    case 5: return launch_p8<T, 5>(p, num_seqs, max_seqlen_q, stream);
    case 6: return launch_p8<T, 6>(p, num_seqs, max_seqlen_q, stream);
    case 7: return launch_p8<T, 7>(p, num_seqs, max_seqlen_q, stream);
    case 8: return launch_p8<T, 8>(p, num_seqs, max_seqlen_q, stream);
  }
  return cudaErrorInvalidValue;
}

template <typename T, int NB>
cudaError_t launch_redo(const CodedPrefillParams &p, cudaStream_t stream) {
  using C = P8Cfg<T, NB>;
  auto kern = fp8_prefill_redo_kernel<T, NB>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  const int ctas = sm_count_current();
  return launch_pdl(kern, dim3(ctas), dim3(kThreads), C::kSmem, stream, p, FastDiv(p.num_q_heads / p.num_kv_heads),
                    FastDiv(p.block_size / kF8Group), ctas);
}

template <typename T>
cudaError_t launch_redo_gathered(const CodedPrefillParams &p, int64_t max_seqlen_q, cudaStream_t stream) {
  using C = P8Cfg<T, 4>;  // the dense kernel has one head_dim
  auto kern = fp8_prefill_redo_gathered_kernel<T, 4>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  const int64_t tiles = (max_seqlen_q * (p.num_q_heads / p.num_kv_heads) + kRows - 1) / kRows;
  int64_t ctas = 2 * sm_count_current() / (p.num_kv_heads * p.num_seqs);
  ctas = ctas < 1 ? 1 : ctas > tiles ? tiles : ctas;
  return launch_pdl(kern, dim3(static_cast<unsigned>(ctas), p.num_kv_heads, static_cast<unsigned>(p.num_seqs)), dim3(kThreads),
                    C::kSmem, stream, p, FastDiv(p.num_q_heads / p.num_kv_heads), FastDiv(p.block_size / kF8Group),
                    static_cast<int>(tiles));
}

}  // namespace

// Splits over the keys: enough CTAs for two per SM, each split at least 256 keys of a full table.
int fp8_prefill_splits(int64_t num_seqs, int64_t max_seqlen_q, int num_q_heads, int num_kv_heads, int64_t capacity,
                       int sms) {
  const int64_t rows = max_seqlen_q * (num_q_heads / num_kv_heads);
  const int64_t ctas = (rows + kRows - 1) / kRows * num_kv_heads * num_seqs;
  int64_t s = 2 * sms / ctas;
  const int64_t most = capacity / 256;
  if (s > most) s = most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}

cudaError_t launch_fp8_prefill(const CodedPrefillParams &p, int dtype, int head_dim, int64_t num_seqs,
                               int64_t max_seqlen_q, cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16) return launch_p8_t<__nv_bfloat16>(p, head_dim, num_seqs, max_seqlen_q, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_p8_t<__half>(p, head_dim, num_seqs, max_seqlen_q, stream);
  return launch_p8_t<float>(p, head_dim, num_seqs, max_seqlen_q, stream);
}

cudaError_t launch_fp8_prefill_redo(const CodedPrefillParams &p, int dtype, int head_dim, cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16)
    return head_dim == 64 ? launch_redo<__nv_bfloat16, 2>(p, stream) : launch_redo<__nv_bfloat16, 4>(p, stream);
  return head_dim == 64 ? launch_redo<__half, 2>(p, stream) : launch_redo<__half, 4>(p, stream);
}

cudaError_t launch_fp8_prefill_redo_gathered(const CodedPrefillParams &p, int dtype, int64_t max_seqlen_q, cudaStream_t stream) {
  return dtype == MI_DTYPE_BFLOAT16 ? launch_redo_gathered<__nv_bfloat16>(p, max_seqlen_q, stream)
                                    : launch_redo_gathered<__half>(p, max_seqlen_q, stream);
}

}  // namespace mi
