// Causal chunked prefill straight from the 4-bit cache (layout: mxfp4.cuh) on
// the warp-level tensor cores, for what the dense tcgen05 kernel behind the gather does
// not take (head_dim other than 128, fp32, other groups) and for chunks too small to fill it.
//
// A CTA takes 128 rows of one kv head, a row being (token, query head of the group), so any group
// fills the tiles; 8 warps of 16 rows.  It walks the keys 64 at a time: codes and scales of
// the next tile are on their way in registers while this one is worked on, then become
// 16-bit K and V rows in the other half of shared memory, decoded once for the 8 warps.  S = Q K^T and
// O += P V are m16n8k16 with fp32 accumulators, P passes from the one to the
// other in registers; online softmax in fp32, the maximum followed 3 binades behind at most.
// Types: bf16 holds every value of the cache (short of overflow), fp16 rounds
// what lies below its smallest step; p in fp16 is lifted by 2^12, which keeps a key down to 2^-26 of
// the largest at full precision.  fp32: K and V are exact in bf16, q and p go in as three bf16 parts
// (24 bits), three MMAs for one.
// A NaN block of V is held as zero and its dims are set to NaN in the rows that
// see the key, so it never reaches rows before it.  So are blocks of K and V that fp16 does not hold, and their products
// are added in fp32, K's to the scores and V's to those rows.
// Few rows over a long context are split over the keys; a second launch joins
// the splits.
// Sums of p V are divided by l at the end, p up to 8 (2^15 in fp16), so V has to stay below 2^127 / (8 * context).
// Measured (bf16): 2048 tokens on 14336, 32/8 heads of 128: 2391 us, 216 TFLOP/s; 8 x 250 on 2000, 16/8
// heads of 64: 93 us, 187 TFLOP/s, of 256: 361 us, 193; fp32, of 128: 362 us, 96.  mma.sync with its operands in
// registers reaches 555 TFLOP/s; what bounds this is latency, 16 warps an SM (128 registers a thread) meeting at a
// barrier per tile (tensor pipe 38% busy, issue slots 43%, 1.7 instructions a cycle, at 8 x 250, heads of 64).
// What it took, 2048 on 6144, 32/8 heads of 64: pages looked up a tile ahead (116 to 110 us at 8 x 250);
// a branch of its own for masked tiles (762 to 651); chunks of 16 bytes a thread, not words (595).
// 32 rows a warp, which halves the reads of K and V fragments, leaves 8 warps and was slower (786 against 762).
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "params.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kRows = 128;
constexpr int kThreads = 256;
constexpr int kKeys = 64;  // keys of a tile
constexpr int kGroups = kKeys / kMxGroup;

template <typename T, int NB>
struct PfCfg {
  static constexpr bool kSplit = std::is_same<T, float>::value;
  using E = typename std::conditional<kSplit, __nv_bfloat16, T>::type;  // MMA operands
  static constexpr int kParts = kSplit ? 3 : 1;
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr uint32_t kApart = mx_apart_from<T>;  // scale bytes from here on are not for the MMA (of K in fp16 alone)
  static constexpr int kMarks = kHalf ? 2 : 1;  // operands with such blocks: V, K
  static constexpr int D = NB * kMxBlock;
  static constexpr int kRowBytes = (NB + 1) / 2 * 128;  // rows of whole 128 bytes, for the swizzle
  static constexpr int kTile = kKeys * kRowBytes;      // K or V of a tile
  static constexpr int kQuery = kRows * kRowBytes;     // one part of q
  static constexpr int kChunks = 2 * kKeys * NB;  // a tile's (operand, key, block): 16 bytes of codes and a scale
  static constexpr int kPer = (kChunks + kThreads - 1) / kThreads;  // of those per thread
  static constexpr int kSmem = kParts * kQuery + 4 * kTile + 2 * (kMarks * kKeys + 4 * kGroups);
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// Byte offset of 16-byte chunk c of a row, chunks swizzled so that 8 rows' reads of one chunk touch every bank.
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
template <typename E>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<E, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename E>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<E, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// What a value leaves after its rounding to E.
template <typename E>
__device__ __forceinline__ float rest(float x) {
  return x - Elem<E>::to_float(Elem<E>::from_float(x));
}

// fp16: rows `row` and row + 8 of q times the blocks of one key that fp16 does not hold, over the four lanes of a row,
// each of which takes 8 dims of a block.  Called among what masked tiles do (a branch of its own after the products took 192 us at
// 8 x 250 on 2000, 16/8 heads of 96, where this takes 172).
template <int NB>
__device__ __noinline__ float2 apart_scores(const uint8_t *codes, unsigned blocks, int tok, const uint8_t *q, int row, int t) {
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
  for (int b = 0; b < NB; ++b) {
    if (!(blocks >> b & 1u)) continue;
    float k8[8];
    mx_codes_to_f32(*reinterpret_cast<const uint32_t *>(codes + b * kMxBlockBytes + tok * 16 + t * 4),
                    mx_scale(codes[NB * kMxBlockBytes + tok * NB + b]), k8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 f[4];
      Vec16<__half>::unpack(*reinterpret_cast<const uint4 *>(q + at<NB>(row + 8 * i, b * 4 + t)), f);
      float &to = i ? sum.y : sum.x;
#pragma unroll
      for (int u = 0; u < 4; ++u) to = fmaf(f[u].x, k8[2 * u], fmaf(f[u].y, k8[2 * u + 1], to));
    }
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) sum.x += __shfl_xor_sync(kAll, sum.x, off), sum.y += __shfl_xor_sync(kAll, sum.y, off);
  return sum;
}

}  // namespace

// 128 rows of one kv head against the keys of one split.
template <typename T, int NB>
__device__ __forceinline__ void prefill_tile(const CodedPrefillParams &p, const FastDiv &by_group, const FastDiv &by_page,
                                             int seq, int kvh, int tile, int split) {
  using C = PfCfg<T, NB>;
  using E = typename C::E;
  constexpr int D = C::D, kParts = C::kParts;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *tiles = smem + kParts * C::kQuery;  // [2][K, V]
  uint8_t *marks = tiles + 4 * C::kTile;  // [2][V, K][keys]: blocks that are not for the MMA, a bit each
  int *group_ok = reinterpret_cast<int *>(marks + 2 * C::kMarks * kKeys);  // [2][groups]
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

  // q into shared memory, as `kParts` operands
  for (int i = threadIdx.x; i < kRows * (D / 8); i += kThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = 0.f;
    const uint32_t row = static_cast<uint32_t>(row0) + r;
    const int64_t token = q0 + by_group.div(row);
    if (r < rows && token >= 0 && token < p.num_tokens) {
      const T *src = static_cast<const T *>(p.query) +
                     (token * p.num_q_heads + kvh * G + (row - by_group.div(row) * G)) * D + c * 8;
      if constexpr (C::kSplit) {
        const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
      } else {
        float2 f[4];
        Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(src), f);
#pragma unroll
        for (int u = 0; u < 4; ++u) x[2 * u] = f[u].x, x[2 * u + 1] = f[u].y;
      }
    }
    // q goes in with the sign of the scale, so that the largest product is the largest score; a scale of 0 or NaN makes it
    // that, and so every score
    if (!(p.scale_log2 > 0.f))
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] *= p.scale_log2 < 0.f ? -1.f : p.scale_log2;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      *reinterpret_cast<uint4 *>(smem + part * C::kQuery + at<NB>(r, c)) =
          make_uint4(pack<E>(x[0], x[1]), pack<E>(x[2], x[3]), pack<E>(x[4], x[5]), pack<E>(x[6], x[7]));
      if (part + 1 < kParts)
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = rest<E>(x[u]);
    }
  }

  // A thread's chunks of a tile, in the order of memory: K's, then V's, (group, block, token).
  struct Words {
    uint4 codes[C::kPer];
    uint32_t scales[C::kPer];  // the scale byte, then whether the page is one
  };
  struct Chunk {
    bool exists, value;
    int group, b;
  };
  auto chunk = [&](int i) {
    const int id = i * kThreads + static_cast<int>(threadIdx.x);
    Chunk c;
    c.exists = C::kChunks % kThreads == 0 || id < C::kChunks;
    c.value = id >= C::kChunks / 2;
    const int gb = (c.value ? id - C::kChunks / 2 : id) / kMxGroup;
    c.group = gb / NB, c.b = gb % NB;
    return c;
  };
  const int per_page = p.block_size / kMxGroup;
  const int32_t *table = p.block_tables + seq * p.bt_stride;
  const int tok = threadIdx.x % kMxGroup;
  // Pages of a tile's chunks are looked up a tile before their codes: kNone past the keys.
  constexpr int kNone = INT32_MIN;
  int pages_at[C::kPer];
  auto look_up = [&](int kt) {
#pragma unroll
    for (int i = 0; i < C::kPer; ++i) {
      const Chunk c = chunk(i);
      const uint32_t index = static_cast<uint32_t>(kt) * kGroups + c.group;
      pages_at[i] = kNone;
      if (c.exists && static_cast<int>(index) * kMxGroup + tok < keys)
        pages_at[i] = max(-1, __ldg(table + by_page.div(index)));
    }
  };
  auto fetch = [&](int kt, Words &w) {
#pragma unroll
    for (int i = 0; i < C::kPer; ++i) {
      const Chunk c = chunk(i);
      const int page = pages_at[i];
      w.codes[i] = make_uint4(0u, 0u, 0u, 0u);
      w.scales[i] = page == kNone ? 1u << 16 : 0u;  // keys that do not exist: zeros
      if (page < 0 || page >= p.num_blocks) continue;
      const uint32_t index = static_cast<uint32_t>(kt) * kGroups + c.group;
      const uint8_t *from = (c.value ? p.value_pages : p.key_pages) +
                            ((static_cast<int64_t>(page) * p.num_kv_heads + kvh) * per_page +
                             (index - by_page.div(index) * per_page)) *
                                (NB * kMxBytes);
      w.codes[i] = *reinterpret_cast<const uint4 *>(from + c.b * kMxBlockBytes + tok * 16);
      w.scales[i] = from[NB * kMxBlockBytes + tok * NB + c.b] | 1u << 16;
    }
  };
  auto place = [&](const Words &w, int buf) {
#pragma unroll
    for (int i = 0; i < C::kPer; ++i) {
      const Chunk c = chunk(i);
      if (!c.exists) continue;
      uint8_t *to = tiles + (buf * 2 + c.value) * C::kTile;
      const int key = c.group * kMxGroup + tok;
      const uint32_t byte = w.scales[i] & 255u;
      const float f = mx_apart<T>(c.value, byte) ? 0.f : mx_scale(byte);
      const uint32_t word[4] = {w.codes[i].x, w.codes[i].y, w.codes[i].z, w.codes[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[8];
        mx_codes_to_f32(word[j], f, x);
        *reinterpret_cast<uint4 *>(to + at<NB>(key, c.b * 4 + j)) =
            make_uint4(pack<E>(x[0], x[1]), pack<E>(x[2], x[3]), pack<E>(x[4], x[5]), pack<E>(x[6], x[7]));
      }
      if (tok == 0 && c.b == 0 && !c.value) {
        const bool ok = (w.scales[i] >> 16) != 0;
        group_ok[buf * kGroups + c.group] = ok;
        if (!ok) flag_status(p.status, MI_DEV_BAD_BLOCK);
      }
    }
  };
  // NaN blocks of V, and those of K and V that fp16 does not hold
  auto note_apart = [&](const Words &w, int buf) -> bool {
    bool any = false;
#pragma unroll
    for (int i = 0; i < C::kPer; ++i) any |= (C::kHalf || chunk(i).value) && (w.scales[i] & 255u) >= C::kApart;
    if (threadIdx.x < C::kMarks * kKeys) marks[buf * C::kMarks * kKeys + threadIdx.x] = 0;
    return any;
  };
  auto mark_apart = [&](const Words &w, int buf) {
#pragma unroll
    for (int i = 0; i < C::kPer; ++i) {
      const Chunk c = chunk(i);
      const int key = c.group * kMxGroup + tok;
      if (c.exists && mx_apart<T>(c.value, w.scales[i] & 255u))
        atomicOr(reinterpret_cast<unsigned *>(marks + (buf * C::kMarks + !c.value) * kKeys) + key / 4,
                 1u << (key % 4 * 8 + c.b));
    }
  };
  // the group of a marked key of tile kt, which has a page
  auto group_of = [&](const uint8_t *pool, int kt, int key) {
    const uint32_t index = static_cast<uint32_t>(kt) * kGroups + key / kMxGroup, col = by_page.div(index);
    return pool + ((static_cast<int64_t>(__ldg(table + col)) * p.num_kv_heads + kvh) * per_page + (index - col * per_page)) *
                      (NB * kMxBytes);
  };

  // this thread's rows: g and g + 8 of its warp's 16
  int pos[2];  // positions are below 2^31 as contexts are
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = warp * 16 + g + 8 * i;
    pos[i] = r < rows ? static_cast<int>(prefix + by_group.div(static_cast<uint32_t>(row0) + r)) : -1;
  }
  const int first_pos = static_cast<int>(prefix + by_group.div(static_cast<uint32_t>(row0) + min(warp * 16, rows - 1)));
  // m follows the largest score, up to kLag binades behind it: p <= 2^(kLift + kLag) is within f16
  const float scale = fabsf(p.scale_log2) > 0.f ? fabsf(p.scale_log2) : 1.f;  // 0 and NaN are in q
  constexpr float kLift = std::is_same<E, __half>::value ? 12.f : 0.f, kLag = 3.f;
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  bool has_apart = false;
  if (k_begin < k_end) {
    Words w;
    look_up(k_begin);
    fetch(k_begin, w);
    look_up(k_begin + 1);
    place(w, 0);
    const bool mine = note_apart(w, 0);
    has_apart = __syncthreads_or(mine);
    if (has_apart) {
      mark_apart(w, 0);
      __syncthreads();
    }
  }
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
    Words w;
    const bool more = kt + 1 < k_end;
    if (more) {
      fetch(kt + 1, w);
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
      for (int part = 0; part < kParts; ++part)
        ldsm(even_chunk(q_lane, ks) + part * C::kQuery, a[part]);
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {  // 16 keys: dims lo, hi of keys 0-7, then of keys 8-15
        uint32_t b[4];
        ldsm(even_chunk(k_base, ks) + n * 16 * C::kRowBytes, b);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          mma<E>(s[2 * n], a[part], b[0], b[1]);
          mma<E>(s[2 * n + 1], a[part], b[2], b[3]);
        }
      }
    }
    const int key0 = kt * kKeys;
    bool pages = true;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) pages &= group_ok[buf * kGroups + i] != 0;
    const bool masked = key0 + kKeys - 1 > first_pos || key0 + kKeys > keys || !pages || (C::kHalf && has_apart);  // uniform in the warp
    if (masked) {
      if constexpr (C::kHalf) {
        if (has_apart) {  // K's blocks past fp16
#pragma unroll 1
          for (int key = 0; key < kKeys; ++key) {
            const unsigned blocks = marks[(buf * C::kMarks + 1) * kKeys + key];
            if (!blocks) continue;
            const float2 sum = apart_scores<NB>(group_of(p.key_pages, kt, key), blocks, key % kMxGroup, smem, warp * 16 + g, t);
            if (t == key % 8 / 2) {
#pragma unroll
              for (int i = 0; i < kKeys / 8; ++i)
                if (i == key / 8) {
                  if (key & 1)
                    s[i][1] += sum.x, s[i][3] += sum.y;
                  else
                    s[i][0] += sum.x, s[i][2] += sum.y;
                }
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
        const int key = key0 + i * 8 + 2 * t;
        const bool none = !group_ok[buf * kGroups + i / 2];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (key + (u & 1) > min(pos[u >> 1], keys - 1) || none) s[i][u] = -INFINITY;
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) top[u >> 1] = fmaxf(top[u >> 1], s[i][u]);
    top[0] *= scale, top[1] *= scale;
    if (__any_sync(kAll, top[0] > m[0] + kLag || top[1] > m[1] + kLag)) {
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
    float base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) base[i] = m[i] == -INFINITY ? 0.f : kLift - m[i];  // no key yet: exp2(-inf) = 0
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s[i][u] = fast_exp2(fmaf(s[i][u], scale, base[u >> 1]));
        // m is off by a step of fp32, which from 2^24 on is binades: p stays within f16, in the sum as in the product
        if constexpr (kLift > 0.f) s[i][u] = fmin_nan(s[i][u], 65504.f);
        l[u >> 1] += s[i][u];
      }
#pragma unroll
    for (int ks = 0; ks < kKeys / 16; ++ks) {
      uint32_t a[kParts][4];
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          a[part][2 * u] = pack<E>(s[2 * ks + u][0], s[2 * ks + u][1]);
          a[part][2 * u + 1] = pack<E>(s[2 * ks + u][2], s[2 * ks + u][3]);
          if (part + 1 < kParts)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[2 * ks + u][c] = rest<E>(s[2 * ks + u][c]);
        }
      }
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {  // 16 dims: keys lo, hi of dims 0-7, then of dims 8-15
        uint32_t b[4];
        ldsm_t(even_chunk(v_base, n) + ks * 16 * C::kRowBytes, b);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          mma<E>(o[2 * n], a[part], b[0], b[1]);
          mma<E>(o[2 * n + 1], a[part], b[2], b[3]);
        }
      }
    }
    if (has_apart) {  // uniform in the CTA
#pragma unroll 1
      for (int key = 0; key < kKeys; ++key) {
        const unsigned blocks = marks[buf * C::kMarks * kKeys + key];
        if (!blocks) continue;
        float pk[2] = {0.f, 0.f};  // p of this key in this thread's rows
        const uint8_t *codes = nullptr;
        if constexpr (C::kHalf) {
#pragma unroll
          for (int i = 0; i < kKeys / 8; ++i)
            if (i == key / 8) pk[0] = key & 1 ? s[i][1] : s[i][0], pk[1] = key & 1 ? s[i][3] : s[i][2];
          pk[0] = __shfl_sync(kAll, pk[0], (lane & ~3) | (key % 8 / 2));
          pk[1] = __shfl_sync(kAll, pk[1], (lane & ~3) | (key % 8 / 2));
          codes = group_of(p.value_pages, kt, key);
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          if (!(blocks >> (n / 4) & 1u)) continue;
          float v[8];
          v[0] = v[1] = __uint_as_float(0x7fffffffu);
          if constexpr (C::kHalf) {
            const int tok = key % kMxGroup;
            const uint32_t byte = codes[NB * kMxBlockBytes + tok * NB + n / 4];
            if (byte != 255u)
              mx_codes_to_f32(*reinterpret_cast<const uint32_t *>(codes + n / 4 * kMxBlockBytes + tok * 16 + n % 4 * 4) >> (8 * t),
                              mx_scale(byte), v);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (key0 + key <= pos[u >> 1]) o[n][u] = C::kHalf ? fmaf(pk[u >> 1], v[u & 1], o[n][u]) : v[0];
        }
      }
    }
    if (more) {
      place(w, buf ^ 1);
      const bool mine = note_apart(w, buf ^ 1);
      has_apart = __syncthreads_or(mine);
      if (has_apart) {
        mark_apart(w, buf ^ 1);
        __syncthreads();
      }
    }
  }

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
    if (p.num_splits == 1) {
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      T *out = static_cast<T *>(p.out) + at_row * D + 2 * t;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        if constexpr (C::kSplit)
          *reinterpret_cast<float2 *>(out + n * 8) = make_float2(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
        else
          *reinterpret_cast<uint32_t *>(out + n * 8) = pack<E>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
      }
    } else {
      float *st = p.workspace + (split * p.num_tokens * p.num_q_heads + at_row) * (D + 2);
      if (t == 0) st[0] = m[i], st[1] = l[i];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2 *>(st + 2 + n * 8 + 2 * t) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    }
  }
}

template <typename T, int NB>
__global__ void __launch_bounds__(kThreads, PfCfg<T, NB>::kSmem <= 100 * 1024 ? 2 : 1)
    mxfp4_prefill_kernel(const CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page) {
  pdl_wait();
  const unsigned at = gridDim.x - 1 - blockIdx.x;  // the last rows, with the most keys, first
  prefill_tile<T, NB>(p, by_group, by_page, blockIdx.z, blockIdx.y, at / p.num_splits, at % p.num_splits);
  pdl_launch_dependents();
}

// After the dense kernel: the sequences and kv heads of which the gather has noted that it cannot do them, over again.  Hardly
// ever any, so a few CTAs look (a CTA to a tile would take 100 us to find nothing at 64 x 2048 tokens) and take all tiles if so.
template <typename T, int NB>
__global__ void __launch_bounds__(kThreads, PfCfg<T, NB>::kSmem <= 100 * 1024 ? 2 : 1)
    mxfp4_prefill_redo_kernel(const CodedPrefillParams p, const FastDiv by_group, const FastDiv by_page, int tiles) {
  pdl_wait();
  const int64_t ctx = static_cast<int64_t>(p.cu_seqlens_k[blockIdx.z + 1]) - p.cu_seqlens_k[blockIdx.z];
  const int64_t groups = min((ctx + kMxGroup - 1) / kMxGroup, static_cast<int64_t>(p.redo_groups));
  const uint8_t *noted = p.redo + (static_cast<int64_t>(blockIdx.z) * p.num_kv_heads + blockIdx.y) * p.redo_stride;
  bool any = false;
  for (int64_t i = threadIdx.x; i < groups; i += kThreads) any |= noted[i] != 0;
  if (__syncthreads_or(any))
    for (int tile = tiles - 1 - blockIdx.x; tile >= 0; tile -= gridDim.x) {
      prefill_tile<T, NB>(p, by_group, by_page, blockIdx.z, blockIdx.y, tile, 0);
      __syncthreads();  // every warp has read its rows of q
    }
  pdl_launch_dependents();
}

// Join the splits: a warp to a row, the rows of the sequences only.
template <typename T, int NB>
__global__ void __launch_bounds__(kThreads) mxfp4_prefill_join_kernel(const CodedPrefillParams p, const FastDiv by_group) {
  constexpr int D = NB * kMxBlock;
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
        L = f * L + e * l;
#pragma unroll
        for (int b = 0; b < NB; ++b) A[b] = f * A[b] + e * a[b];
        M = next;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
        static_cast<T *>(p.out)[at_row * D + b * 32 + lane] = Elem<T>::from_float(L == 0.f ? 0.f : A[b] / L);
    }
  }
  pdl_launch_dependents();
}

namespace {

template <typename T, int NB>
cudaError_t launch_pf(const CodedPrefillParams &p, int64_t num_seqs, int64_t max_seqlen_q, cudaStream_t stream) {
  using C = PfCfg<T, NB>;
  auto kern = mxfp4_prefill_kernel<T, NB>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int G = p.num_q_heads / p.num_kv_heads;
  const int64_t tiles = (max_seqlen_q * G + kRows - 1) / kRows;
  const FastDiv by_group(G), by_page(p.block_size / kMxGroup);
  if constexpr (NB == 4 && !C::kSplit) {
    if (p.redo != nullptr) {
      auto redo = mxfp4_prefill_redo_kernel<T, NB>;
      static bool redo_attr_set[64] = {};
      if (dev >= 64 || !redo_attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(redo, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < 64) redo_attr_set[dev] = true;
      }
      int64_t ctas = 2 * sm_count_current() / (p.num_kv_heads * num_seqs);
      ctas = ctas < 1 ? 1 : ctas > tiles ? tiles : ctas;
      return launch_pdl(redo, dim3(static_cast<unsigned>(ctas), p.num_kv_heads, static_cast<unsigned>(num_seqs)),
                        dim3(kThreads), C::kSmem, stream, p, by_group, by_page, static_cast<int>(tiles));
    }
  }
  if (p.redo != nullptr) return cudaErrorInvalidValue;
  if (dev >= 64 || !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev] = true;
  }
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(tiles * p.num_splits), p.num_kv_heads,
                                        static_cast<unsigned>(num_seqs)),
                             dim3(kThreads), C::kSmem, stream, p, by_group, by_page);
  if (e == cudaSuccess && p.num_splits > 1)
    e = launch_pdl(mxfp4_prefill_join_kernel<T, NB>,
                   dim3(static_cast<unsigned>((max_seqlen_q * G + kThreads / 32 - 1) / (kThreads / 32)),
                        p.num_kv_heads, static_cast<unsigned>(num_seqs)),
                   dim3(kThreads), 0, stream, p, by_group);
  return e;
}

template <typename T>
cudaError_t launch_pf_t(const CodedPrefillParams &p, int head_dim, int64_t num_seqs, int64_t max_seqlen_q,
                        cudaStream_t stream) {
  switch (head_dim / kMxBlock) {
    case 1: return launch_pf<T, 1>(p, num_seqs, max_seqlen_q, stream);
    case 2: return launch_pf<T, 2>(p, num_seqs, max_seqlen_q, stream);
    case 3: return launch_pf<T, 3>(p, num_seqs, max_seqlen_q, stream);
    case 4: return launch_pf<T, 4>(p, num_seqs, max_seqlen_q, stream);
  }
  if constexpr (!std::is_same<T, float>::value) {
    switch (head_dim / kMxBlock) {
      case 5: return launch_pf<T, 5>(p, num_seqs, max_seqlen_q, stream);
      case 6: return launch_pf<T, 6>(p, num_seqs, max_seqlen_q, stream);
      case 7: return launch_pf<T, 7>(p, num_seqs, max_seqlen_q, stream);
      case 8: return launch_pf<T, 8>(p, num_seqs, max_seqlen_q, stream);
    }
  }
  return cudaErrorInvalidValue;
}

}  // namespace

// Shared memory holds q's three parts in fp32 up to head_dim 128.
bool mxfp4_prefill_supported(int dtype, int head_dim) {
  return head_dim % kMxBlock == 0 && head_dim <= (dtype == MI_DTYPE_FLOAT32 ? 128 : 256);
}

// Splits over the keys: enough CTAs for two per SM, each split at least 4 tiles of a full table.
int mxfp4_prefill_splits(int64_t num_seqs, int64_t max_seqlen_q, int num_q_heads, int num_kv_heads,
                         int64_t capacity, int sms) {
  const int64_t rows = max_seqlen_q * (num_q_heads / num_kv_heads);
  const int64_t ctas = (rows + kRows - 1) / kRows * num_kv_heads * num_seqs;
  int64_t s = 2 * sms / ctas;
  const int64_t most = capacity / (4 * kKeys);
  if (s > most) s = most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}

cudaError_t launch_mxfp4_prefill(const CodedPrefillParams &p, int dtype, int head_dim, int64_t num_seqs,
                                 int64_t max_seqlen_q, cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16) return launch_pf_t<__nv_bfloat16>(p, head_dim, num_seqs, max_seqlen_q, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_pf_t<__half>(p, head_dim, num_seqs, max_seqlen_q, stream);
  return launch_pf_t<float>(p, head_dim, num_seqs, max_seqlen_q, stream);
}

}  // namespace mi
