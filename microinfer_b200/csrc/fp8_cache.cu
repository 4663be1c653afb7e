// Moving K and V into and out of the 8-bit paged cache (layout: fp8.cuh).
//
// Store.  The tokens of a call that fall into one group (16 slots of a kv head) are quantised together: with a their largest
// finite magnitude they need the scale 2^e, e the least exponent with a <= 448 * 2^e.  A call that writes the group's
// first slot sets the scale to that (the group starts anew); any other raises it to that at most, and where it rises by 2^s
// the group's other codes are divided by 2^s, rounded once.  So a sequence that grows token by token re-rounds a code
// only where its value is subnormal, and a page's last owner leaves nothing behind.
//
// Which tokens share a group is not in the order of the slots (a batch's rows may come in any), and a group must have one
// writer.  The first token of a group in the call's order is its owner.  Short calls: a CTA per token, whose threads look through
// all slots for the token's group.  Longer ones: a launch before it writes each token's number to index[slot],
// and a CTA of up to 256 tokens reads the 16 entries of each of their groups; the index needs no initial value, since an
// entry i is this call's where slots[i] is the slot again.
// An owner's rows are read at once (8 16-byte loads a lane at head_dim 128 in 16 bits): the maximum goes through five
// shuffles and the codes are written from registers, whole 32-byte sectors of K and V.
//
// Gather: rows of each request in logical order, request-major, as code * scale in the requested type (exact in fp32 and
// bf16; fp16 rounds).  A warp takes a group of 16 positions of one kv head and writes 16 bytes a lane, whole rows together.
// HBM-bound on the rows that it writes.
//
// Measured, 8 heads of 128: store of 32 tokens 4.6 us, 8000 in bf16 18 and in fp32 29, 64000 in bf16 75 (5.3 TB/s, 80% of a copy; issue
// slots 62%, ALU 50%); scan and index, us: 300 tokens 8 : 11, 1000 14 : 13,
// 2000 22 : 13; where each token has a group of its own 300 12 : 15, 1000 25 : 26, 2000 45 : 38.  Gather of 48 x 1500 to bf16 69 us (5.6 TB/s).
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.cuh"
#include "params.cuh"

namespace mi {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kChunk = 256;      // tokens of a CTA that finds groups by the index, at most
constexpr int kScanTokens = 512; // calls up to this long look through the slots instead, without an index

// Eight elements of a row as they are in memory.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *src, Raw8<T> &r) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4 *>(src)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T *>(r.v)[i] = src[i];
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
    constexpr int N = Vec16<T>::N;
    float2 f[N / 2];
    Vec16<T>::unpack(r.v[i], f);
#pragma unroll
    for (int u = 0; u < N / 2; ++u) x[N * i + 2 * u] = f[u].x, x[N * i + 2 * u + 1] = f[u].y;
  }
}

__device__ __forceinline__ int64_t slot_at(const CodedStoreParams &p, int64_t t) {
  return p.wide_slots ? static_cast<const int64_t *>(p.slots)[t] : static_cast<const int32_t *>(p.slots)[t];
}

__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inverse) {
  float y[8];  // x - x: NaN for an infinity, which the conversion would make 448; else -0, which keeps the sign of a zero
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fmaf(x[i], inverse, -(x[i] - x[i]));
  return make_uint2(f8_encode4(y[0], y[1], y[2], y[3]), f8_encode4(y[4], y[5], y[6], y[7]));
}

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float factor) {
  float x[4];
  f8_to_f32(w, x);
  return f8_encode4(x[0] * factor, x[1] * factor, x[2] * factor, x[3] * factor);
}

// V's bytes of two tokens from each one's codes of 8 dims, and back.
__device__ __forceinline__ uint4 interleave(uint2 a, uint2 b) {
  return make_uint4(__byte_perm(a.x, b.x, 0x5140), __byte_perm(a.x, b.x, 0x7362), __byte_perm(a.y, b.y, 0x5140),
                    __byte_perm(a.y, b.y, 0x7362));
}
__device__ __forceinline__ void separate(uint4 v, uint2 &a, uint2 &b) {
  a = make_uint2(__byte_perm(v.x, v.y, 0x6420), __byte_perm(v.z, v.w, 0x6420));
  b = make_uint2(__byte_perm(v.x, v.y, 0x7531), __byte_perm(v.z, v.w, 0x7531));
}
// WHOLE: the 16 bytes of 8 dims of a pair lie together.
template <bool WHOLE>
__device__ __forceinline__ uint4 read_pair(const uint8_t *at, int split) {
  if constexpr (WHOLE) return *reinterpret_cast<const uint4 *>(at);
  const uint2 lo = *reinterpret_cast<const uint2 *>(at), hi = *reinterpret_cast<const uint2 *>(at + split);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}
template <bool WHOLE>
__device__ __forceinline__ void write_pair(uint8_t *at, int split, uint4 v) {
  if constexpr (WHOLE) {
    *reinterpret_cast<uint4 *>(at) = v;
    return;
  }
  *reinterpret_cast<uint2 *>(at) = make_uint2(v.x, v.y);
  *reinterpret_cast<uint2 *>(at + split) = make_uint2(v.z, v.w);
}

// index[slot] = the token that goes there.
__global__ void __launch_bounds__(256) fp8_index_kernel(const CodedStoreParams p) {
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t < p.num_tokens) {
    const int64_t slot = slot_at(p, t);
    if (slot >= 0 && slot < p.num_slots) p.index[slot] = static_cast<int32_t>(t);
  }
  pdl_launch_dependents();
}

// One operand's tokens of a group and kv head, by a warp.  member[j]: the token that goes to slot j of the group, or -1.
// NB blocks of 32 dims, whose rows stay in registers; 0: any number, read twice.
template <typename T, bool VEC, int NB, bool VALUE>
__device__ __forceinline__ void store_group(const CodedStoreParams &p, uint8_t *group, const int32_t *member, int head, int lane) {
  const int D = NB > 0 ? NB * 32 : p.head_dim, items = D / 32, octets = D / 8;
  const T *rows = static_cast<const T *>(VALUE ? p.values : p.keys) + head * D;
  const int64_t stride = VALUE ? p.value_stride : p.key_stride;
  const bool fresh = member[0] >= 0;
  const uint32_t old = fresh ? 0u : group[kF8Group * D];
  constexpr int kHeld = NB > 0 ? NB : 1;
  constexpr bool kWhole = NB > 0 && NB % 2 == 0;
  Raw8<T> x[kHeld][2];
  // item i of a lane: 8 dims of a pair of tokens
  auto pair_of = [&](int i) { return (i * 32 + lane) / octets; };
  auto octet_of = [&](int i) { return (i * 32 + lane) % octets; };
  auto read = [&](int i, Raw8<T> (&v)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = member[2 * pair_of(i) + k];
      v[k] = Raw8<T>{};
      if (t >= 0) load8<T, VEC>(rows + t * stride + octet_of(i) * 8, v[k]);
    }
  };
  // Largest magnitude as bits of T, which order like the values with NaN above infinity; 16-bit ones two to a word, never
  // unpacked for it.  Where something is not finite, once more without that.
  constexpr uint32_t kMask = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  constexpr uint32_t kInf = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  uint32_t top = 0;
  auto larger = [](uint32_t u, uint32_t v) { return sizeof(T) == 2 ? __vmaxu2(u, v) : max(u, v); };
  auto look = [&](const Raw8<T> (&v)[2], bool finite) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        const uint32_t w[4] = {v[k].v[i].x, v[k].v[i].y, v[k].v[i].z, v[k].v[i].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t bits = w[u] & kMask;
          if (finite) bits &= sizeof(T) == 2 ? __vcmpltu2(bits, kInf) : bits < kInf ? ~0u : 0u;
          top = larger(top, bits);
        }
      }
  };
  if constexpr (NB > 0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) read(i, x[i]);
#pragma unroll
    for (int i = 0; i < NB; ++i) look(x[i], false);
    const bool all = sizeof(T) == 2 ? __vcmpltu2(top, kInf) == ~0u : top < kInf;
    if (__any_sync(kAll, !all)) {
      top = 0;
#pragma unroll
      for (int i = 0; i < NB; ++i) look(x[i], true);
    }
  } else {
    for (int i = 0; i < items; ++i) {
      read(i, x[0]);
      look(x[0], true);
    }
  }
  if constexpr (sizeof(T) == 2) {
    const uint16_t most = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    top = __float_as_uint(Elem<T>::to_float(*reinterpret_cast<const T *>(&most)));
  }
  const uint32_t need = f8_byte_for(__reduce_max_sync(kAll, top));
  const uint32_t byte = max(need, old);
  const bool grown = !fresh && byte > old;
  const float inverse = byte == 0 ? 1.f : __uint_as_float((254u - byte) << 23);
  const float factor = old == 0 || byte - old > 126u ? 0.f : __uint_as_float((127u + old - byte) << 23);
  auto write = [&](int i, const Raw8<T> (&v)[2]) {
    const int pair = pair_of(i);
    const F8Place at = f8_place(octet_of(i), D);
    bool in[2];
    uint2 w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      in[k] = member[2 * pair + k] >= 0;
      float f[8];
      unpack8(v[k], f);
      w[k] = encode8(f, inverse);
    }
    if constexpr (VALUE) {
      if (!in[0] && !in[1] && !grown) return;
      uint8_t *to = group + at.v + (pair >> 2) * at.half + (pair & 3) * at.pair;
      if (!(in[0] && in[1])) {
        uint2 was[2];
        separate(read_pair<kWhole>(to, at.split), was[0], was[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (in[k]) continue;
          w[k] = grown ? make_uint2(rescale4(was[k].x, factor), rescale4(was[k].y, factor)) : was[k];
        }
      }
      write_pair<kWhole>(to, at.split, interleave(w[0], w[1]));
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint2 *to = reinterpret_cast<uint2 *>(group + at.k + (2 * pair + k) * at.row);
        if (!in[k]) {
          if (!grown) continue;
          const uint2 was = *to;
          w[k] = make_uint2(rescale4(was.x, factor), rescale4(was.y, factor));
        }
        *to = w[k];
      }
    }
  };
  if constexpr (NB > 0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) write(i, x[i]);
  } else {
    for (int i = 0; i < items; ++i) {
      read(i, x[0]);
      write(i, x[0]);
    }
  }
  __syncwarp();  // every lane has read the old byte
  if (lane == 0 && (fresh || grown)) group[kF8Group * D] = static_cast<uint8_t>(byte);
}

// 128-byte lines of one operand's row of a head, into L2.
template <typename T>
__device__ __forceinline__ void prefetch_row(const T *row, int head_dim, int part, int parts) {
  const char *from = reinterpret_cast<const char *>(row);
  for (int at = part * 128; at < head_dim * static_cast<int>(sizeof(T)); at += parts * 128)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(from + at));
}

// A CTA takes one token (SCAN) or `chunk` of them, at most kChunk, and 8 of the kv heads' operands, one to a warp.  Rows are on their
// way into L2 while the CTA finds out where the first of them go, and while the group before theirs is worked on.
template <typename T, bool VEC, int NB, bool SCAN>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) fp8_store_kernel(const CodedStoreParams p, int chunk) {
  constexpr int kTokens = SCAN ? 1 : kChunk;
  __shared__ int32_t member[kTokens][kF8Group];
  __shared__ int64_t owned[kTokens];  // groups of the pool
  __shared__ int num_owned;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int operand = blockIdx.y * 8 + warp, head = operand >> 1;
  const T *rows = static_cast<const T *>(operand & 1 ? p.values : p.keys) + head * p.head_dim;
  const int64_t stride = operand & 1 ? p.value_stride : p.key_stride;
  const int64_t first = SCAN ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * chunk;
  if (head < p.num_kv_heads) {
    const int64_t t = first + (lane >> 1);
    if (t < p.num_tokens && (lane >> 1) < chunk) prefetch_row(rows + t * stride, p.head_dim, lane & 1, 2);
  }
  pdl_wait();
  if constexpr (SCAN) {
    if (threadIdx.x < kF8Group) member[0][threadIdx.x] = -1;
    const int64_t slot = slot_at(p, first);
    const bool good = slot >= 0 && slot < p.num_slots;
    if (!good && slot != -1 && threadIdx.x == 0) flag_status(p.status, MI_DEV_BAD_SLOT);
    __syncthreads();
    bool earlier = false;
    if (good)
      for (int i = threadIdx.x; i < p.num_tokens; i += blockDim.x) {
        const int64_t s = slot_at(p, i);
        if (s >= 0 && s / kF8Group == slot / kF8Group) {
          atomicMax(&member[0][s % kF8Group], i);
          earlier |= i < first;
        }
      }
    if (__syncthreads_or(earlier) || !good) return;
    if (threadIdx.x == 0) num_owned = 1, owned[0] = slot / kF8Group;
  } else {
    if (threadIdx.x == 0) num_owned = 0;
    __syncthreads();
    const int64_t t = first + threadIdx.x;
    const bool mine = threadIdx.x < chunk && t < p.num_tokens;
    const int64_t slot = mine ? slot_at(p, t) : -1;
    const bool good = slot >= 0 && slot < p.num_slots;
    if (!good && slot != -1) flag_status(p.status, MI_DEV_BAD_SLOT);
    if (good) {
      const int64_t base = slot - slot % kF8Group;
      int32_t entry[kF8Group], least = INT32_MAX;
#pragma unroll
      for (int j = 0; j < kF8Group; j += 4) {
        const int4 v = __ldcg(reinterpret_cast<const int4 *>(p.index + base + j));
        entry[j] = v.x, entry[j + 1] = v.y, entry[j + 2] = v.z, entry[j + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < kF8Group; ++j) {
        const bool there = entry[j] >= 0 && entry[j] < p.num_tokens && slot_at(p, entry[j]) == base + j;
        entry[j] = there ? entry[j] : -1;
        if (there) least = min(least, entry[j]);
      }
      if (least == t) {  // the group's first token
        const int at = atomicAdd(&num_owned, 1);
        owned[at] = slot / kF8Group;
#pragma unroll
        for (int j = 0; j < kF8Group; ++j) member[at][j] = entry[j];
      }
    }
  }
  __syncthreads();
  const int per_page = p.block_size / kF8Group, bytes = f8_group_bytes(p.head_dim);
  if (head < p.num_kv_heads)
    for (int i = 0; i < num_owned; ++i) {
      if (i + 1 < num_owned) {
        const int t = member[i + 1][lane >> 1];
        if (t >= 0) prefetch_row(rows + t * stride, p.head_dim, lane & 1, 2);
      }
      const int64_t page = owned[i] / per_page;
      const int64_t at = ((page * p.num_kv_heads + head) * per_page + (owned[i] - page * per_page)) * bytes;
      if (operand & 1)
        store_group<T, VEC, NB, true>(p, p.value_pages + at, member[i], head, lane);
      else
        store_group<T, VEC, NB, false>(p, p.key_pages + at, member[i], head, lane);
    }
  pdl_launch_dependents();
}

template <typename T>
__device__ __forceinline__ void write8(T *dst, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint4 v;
    T *e = reinterpret_cast<T *>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_float(x[i]);
    *reinterpret_cast<uint4 *>(dst) = v;
  } else {
    reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// grid (groups of 16 positions x kv heads, 8 warps to a CTA; sequences).  REDO: rows for the dense prefill, which cannot
// do NaN of V (0 * NaN reaches rows that do not see the key; one of K only meets its own scores) nor values at the ends of
// the range: the sequences and heads that have some are noted.
template <typename T, int NB, bool REDO>
__global__ void __launch_bounds__(256) fp8_gather_kernel(const CodedGatherParams p, const FastDiv by_heads,
                                                         const FastDiv by_page) {
  pdl_wait();
  const int seq = blockIdx.y;
  const int64_t base = p.cu_seqlens_k[seq];
  const int64_t ctx = p.cu_seqlens_k[seq + 1] - base;
  const int lane = threadIdx.x & 31;
  const uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t g = by_heads.div(task);
  const int h = static_cast<int>(task - g * p.num_kv_heads);
  const int64_t pos0 = static_cast<int64_t>(g) * kF8Group;
  if (pos0 >= ctx || (p.fill && g >= p.fill)) return;
  const int D = NB > 0 ? NB * 32 : p.head_dim, items = D / 32, octets = D / 8;
  auto pair_of = [&](int i) { return (i * 32 + lane) / octets; };
  auto octet_of = [&](int i) { return (i * 32 + lane) % octets; };
  bool apart = false;
  auto note = [&] {  // before the warp returns
    if constexpr (REDO) {
      const bool any = __any_sync(kAll, apart);
      if (lane == 0) p.redo[(static_cast<int64_t>(seq) * p.num_kv_heads + h) * p.redo_stride + g] = any;
    }
  };
  auto zero_group = [&](int64_t from) {
    const float zeros[8] = {};
    for (int i = 0; i < items; ++i)
      for (int k = 0; k < 2; ++k) {
        const int64_t pos = from + 2 * pair_of(i) + k, row = base + pos;
        if (pos >= ctx || row < 0 || row >= p.out_rows) continue;
        const int64_t dst = (row * p.num_kv_heads + h) * D + octet_of(i) * 8;
        write8(static_cast<T *>(p.out_keys) + dst, zeros);
        write8(static_cast<T *>(p.out_values) + dst, zeros);
      }
  };
  if (p.fill && ctx > static_cast<int64_t>(p.fill) * kF8Group) {
    if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    apart = true;
    for (int64_t more = g + static_cast<int64_t>(p.fill); more * kF8Group < min(ctx, p.out_rows); more += p.fill)
      zero_group(more * kF8Group);
  }
  const int64_t col = by_page.div(g);  // groups of a page
  const int per_page = p.block_size / kF8Group;
  const int64_t blk = col < p.block_table_stride ? p.block_tables[seq * p.block_table_stride + col] : -1;
  if (blk < 0 || blk >= p.num_blocks) {
    if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    apart = true;  // to be left out, as prefill from the pages does
    if (p.fill) zero_group(pos0);
    note();
    return;
  }
  const int64_t off = ((blk * p.num_kv_heads + h) * per_page + (g - col * per_page)) * f8_group_bytes(D);
  const uint8_t *kg = p.key_pages + off, *vg = p.value_pages + off;
  const uint32_t kbyte = __ldg(kg + kF8Group * D), vbyte = __ldg(vg + kF8Group * D);
  const float ks = f8_scale(kbyte), vs = f8_scale(vbyte);
  // What the dense kernel does not hold.  fp16: values past its range, and of K those that lose bits below its smallest step (of V
  // they are as small in the result).  bf16, whose sums of products meet the softmax's scale behind them: K
  // beyond 2^-64 to 2^64, V above it, whose sums over a long context leave fp32's range.
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const bool far = REDO && kHalf && max(kbyte, vbyte) >= 127u + 8u;         // 448 * 2^7 < 65504
  const bool low = REDO && kHalf && kbyte != 0 && kbyte < 127u + 9u - 24u;  // codes are multiples of 2^-9
  if (REDO && !kHalf) apart |= max(kbyte, vbyte) > 127u + 64u || (kbyte != 0 && kbyte < 127u - 64u);
  constexpr int kHeld = NB > 0 ? NB : 1;
  constexpr bool kWhole = NB > 0 && NB % 2 == 0;
  for (int i0 = 0; i0 < items; i0 += kHeld) {
    uint2 kw[kHeld][2];
    uint4 vw[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {  // every code is in the page: read whether wanted or not
      const F8Place at = f8_place(octet_of(i0 + u), D);
      const int pair = pair_of(i0 + u);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        kw[u][k] = __ldg(reinterpret_cast<const uint2 *>(kg + at.k + (2 * pair + k) * at.row));
      vw[u] = read_pair<kWhole>(vg + at.v + (pair >> 2) * at.half + (pair & 3) * at.pair, at.split);
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      uint2 v[2];
      separate(vw[u], v[0], v[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t pos = pos0 + 2 * pair_of(i0 + u) + k, row = base + pos;
        if (pos >= ctx) continue;
        if (row < 0 || row >= p.out_rows) {
          flag_status(p.status, MI_DEV_BAD_SLOT);
          continue;
        }
        const int64_t dst = (row * p.num_kv_heads + h) * D + octet_of(i0 + u) * 8;
        float x[8], y[8], a[4], b[4];
        f8_to_f32(kw[u][k].x, a);
        f8_to_f32(kw[u][k].y, b);
#pragma unroll
        for (int n = 0; n < 4; ++n) x[n] = a[n] * ks, x[n + 4] = b[n] * ks;
        write8(static_cast<T *>(p.out_keys) + dst, x);
        f8_to_f32(v[k].x, a);
        f8_to_f32(v[k].y, b);
#pragma unroll
        for (int n = 0; n < 4; ++n) y[n] = a[n] * vs, y[n + 4] = b[n] * vs;
        write8(static_cast<T *>(p.out_values) + dst, y);
        if constexpr (REDO) {
          apart |= f8_any_nan(v[k].x) || f8_any_nan(v[k].y);
          if (far)
#pragma unroll
            for (int n = 0; n < 8; ++n) apart |= fmaxf(fabsf(x[n]), fabsf(y[n])) > 65504.f;  // the next one is 65536
          if (low)
#pragma unroll
            for (int n = 0; n < 8; ++n) apart |= __half2float(__float2half_rn(x[n])) != x[n];
        }
      }
    }
  }
  note();
  pdl_launch_dependents();
}

template <typename T, bool VEC, int NB>
cudaError_t launch_store_nb(const CodedStoreParams &p, cudaStream_t stream) {
  const dim3 block(p.num_kv_heads >= 4 ? 256 : 64 * p.num_kv_heads);
  const unsigned operands = static_cast<unsigned>((2 * p.num_kv_heads + 7) / 8);
  if (p.index == nullptr)
    return launch_pdl(fp8_store_kernel<T, VEC, NB, true>, dim3(static_cast<unsigned>(p.num_tokens), operands), block, 0,
                      stream, p, 1);
  const cudaError_t e = launch_pdl(fp8_index_kernel, dim3(static_cast<unsigned>((p.num_tokens + 255) / 256)), dim3(256), 0,
                                   stream, p);
  if (e != cudaSuccess) return e;
  // One round of CTAs, as far as it goes: finding the groups is paid once by each (about 2 us).
  const int64_t ctas = (sizeof(T) == 2 ? 4 : 2) * static_cast<int64_t>(sm_count_current()) / operands;
  int64_t chunk = (p.num_tokens + (ctas > 0 ? ctas : 1) - 1) / (ctas > 0 ? ctas : 1);
  // Below a group's tokens as it is: where each token has a group of its own (a decode step of many sequences) a CTA's
  // are worked on one after the other.
  if (chunk > kF8Group) chunk = (chunk + kF8Group - 1) / kF8Group * kF8Group;
  if (chunk > kChunk) chunk = kChunk;
  if (chunk > static_cast<int64_t>(block.x)) chunk = block.x;  // a thread to a token
  return launch_pdl(fp8_store_kernel<T, VEC, NB, false>,
                    dim3(static_cast<unsigned>((p.num_tokens + chunk - 1) / chunk), operands), block, 0, stream, p,
                    static_cast<int>(chunk));
}

template <typename T, bool VEC>
cudaError_t launch_store_t(const CodedStoreParams &p, cudaStream_t stream) {
  if constexpr (VEC) {
    if (p.head_dim == 128) return launch_store_nb<T, VEC, 4>(p, stream);
    if (p.head_dim == 64) return launch_store_nb<T, VEC, 2>(p, stream);
  }
  return launch_store_nb<T, VEC, 0>(p, stream);
}

template <typename T, bool REDO>
cudaError_t launch_gather_t(const CodedGatherParams &p, int64_t num_seqs, int64_t max_context, cudaStream_t stream) {
  const int64_t tasks = (max_context + kF8Group - 1) / kF8Group * p.num_kv_heads;
  if (tasks >= (int64_t{1} << 31)) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((tasks + 7) / 8), static_cast<unsigned>(num_seqs)), block(256);
  const FastDiv by_heads(p.num_kv_heads), by_page(p.block_size / kF8Group);
  if (p.head_dim == 128)
    return launch_pdl(fp8_gather_kernel<T, 4, REDO>, grid, block, 0, stream, p, by_heads, by_page);
  if constexpr (REDO) return cudaErrorInvalidValue;  // the dense kernel has one head_dim
  if (p.head_dim == 64) return launch_pdl(fp8_gather_kernel<T, 2, false>, grid, block, 0, stream, p, by_heads, by_page);
  return launch_pdl(fp8_gather_kernel<T, 0, false>, grid, block, 0, stream, p, by_heads, by_page);
}

}  // namespace

// Entries of the index that a store of this many tokens needs: a slot's each, or none.
int64_t fp8_store_index_entries(int64_t num_tokens, int64_t num_slots) { return num_tokens <= kScanTokens ? 0 : num_slots; }

cudaError_t launch_fp8_store(const CodedStoreParams &p, int dtype, bool vec, cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16)
    return vec ? launch_store_t<__nv_bfloat16, true>(p, stream) : launch_store_t<__nv_bfloat16, false>(p, stream);
  if (dtype == MI_DTYPE_FLOAT16)
    return vec ? launch_store_t<__half, true>(p, stream) : launch_store_t<__half, false>(p, stream);
  return vec ? launch_store_t<float, true>(p, stream) : launch_store_t<float, false>(p, stream);
}

cudaError_t launch_fp8_gather(const CodedGatherParams &p, int dtype, int64_t num_seqs, int64_t max_context,
                              cudaStream_t stream) {
  if (p.redo != nullptr)
    return dtype == MI_DTYPE_BFLOAT16 ? launch_gather_t<__nv_bfloat16, true>(p, num_seqs, max_context, stream)
                                      : launch_gather_t<__half, true>(p, num_seqs, max_context, stream);
  if (dtype == MI_DTYPE_BFLOAT16) return launch_gather_t<__nv_bfloat16, false>(p, num_seqs, max_context, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_gather_t<__half, false>(p, num_seqs, max_context, stream);
  return launch_gather_t<float, false>(p, num_seqs, max_context, stream);
}

}  // namespace mi
