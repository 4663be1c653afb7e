// Moving K and V into and out of the 4-bit paged cache (layout: mxfp4.cuh).
//
// Store: for each block of 32 elements x with a = max |x|, the scale is
//   2^e, e = floor(log2 a) - 2  (so that a / 2^e lies in [4, 8), the top binade of e2m1),
// held as the byte e + 127, at least 1; codes are x / 2^e rounded to the
// nearest e2m1 value (ties to even, saturating at 6).  The division by a power
// of two is exact, so codes and scales do not depend on the order of any sum.
// A zero block has the byte 0, a block with an infinity or a NaN the byte 255.
// A warp takes 8 consecutive tokens of one kv head, four lanes to a token: a lane loads
// 8 elements of every block of K and V before it uses any, two shuffles give a
// block's a, and the tokens' codes of one block are 128 consecutive bytes, their scales 32 (at
// D = 128) where the slots are consecutive.  Reads 2 or 4 bytes per element and writes 4.25
// bits: HBM-bound on the read, where there is enough of it.  8000 tokens of 8 heads of 128 in bf16: 10.7 us,
// 3.9 TB/s, fp32 15.0 us, 5.0 TB/s (every warp loads, encodes and writes once, with nothing to overlap; the plain
// 16-bit store moves 34 MB at 4.6 TB/s); 64000 tokens 64.6 us, 5.1 TB/s, fp32 90.3 us, 6.6 TB/s; 8 tokens: 2.0 us.
//
// Gather: rows of each request in logical order, request-major, as
// code * scale in the requested type (exact in fp32 and bf16 short of
// overflow; fp16 rounds).  A warp takes a group of 16 positions of one kv head, four lanes to a token as
// above; the heads of a group go to neighbouring warps, which write whole rows
// together.  HBM-bound on the rows that it writes: 64 x 1152 rows of 8 heads of 128 to bf16 in 62 us,
// 6.1 TB/s (95% of the copy rate); to fp32 163 us, 4.2 TB/s.
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "params.cuh"

namespace mi {

namespace {

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
  if constexpr (VEC && sizeof(T) == 2) {
    float2 f[4];
    Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(src), f);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = f[i].x, x[2 * i + 1] = f[i].y;
  } else if constexpr (VEC) {
    const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_float(src[i]);
  }
}

// Quantise 8 of a block's 32 elements (the quad's other lanes hold the rest); returns the codes, `byte`
// the block's scale.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t &byte) {
  uint32_t top = 0;  // largest magnitude as bits: orders like the floats, NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  byte = top >> 23;
  byte = byte > 3 ? byte - 2 : 1;  // the lowest scale is 2^-126
  const float inv = __uint_as_float((254u - byte) << 23);
  uint32_t w = mx_encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv) & 0xffffu;
  w |= mx_encode4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv) << 16;
  if (top == 0) byte = 0;
  if (top >= 0x7f800000u) byte = 255, w = 0;
  return w;
}

// Blocks of a head: the template's, or at run time where that is 0.
template <int NB>
__device__ __forceinline__ int blocks_of(int head_dim) {
  return NB > 0 ? NB : head_dim / kMxBlock;
}

// One warp per (8 tokens, kv head).  WIDE: slots past 32 bits.
template <typename T, typename I, bool VEC, int NB, bool WIDE>
__global__ void __launch_bounds__(128) mxfp4_store_kernel(const MxStoreParams p, const FastDiv by_heads,
                                                          const FastDiv by_block) {
  pdl_wait();
  const int lane = threadIdx.x & 31, j = lane & 3;
  const uint32_t task = blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t chunk = by_heads.div(task);
  const int h = static_cast<int>(task - chunk * p.num_kv_heads);
  const int64_t t = static_cast<int64_t>(chunk) * 8 + (lane >> 2);
  const int nb = blocks_of<NB>(p.head_dim);
  int64_t slot = -1;
  if (t < p.num_tokens) slot = static_cast<int64_t>(static_cast<const I *>(p.slots)[t]);
  if (slot < -1 || slot >= p.num_slots) {
    if (j == 0 && h == 0) flag_status(p.status, MI_DEV_BAD_SLOT);
    slot = -1;
  }
  const T *krow = static_cast<const T *>(p.keys) + t * p.key_stride + h * p.head_dim + j * 8;
  const T *vrow = static_cast<const T *>(p.values) + t * p.value_stride + h * p.head_dim + j * 8;
  int64_t page, offset;
  if constexpr (WIDE) {
    page = (slot < 0 ? 0 : slot) / p.block_size;
    offset = (slot < 0 ? 0 : slot) - page * p.block_size;
  } else {
    const uint32_t s = slot < 0 ? 0 : static_cast<uint32_t>(slot);
    page = by_block.div(s);
    offset = s - static_cast<uint32_t>(page) * p.block_size;
  }
  const int tok = static_cast<int>(offset % kMxGroup);
  const int64_t group = ((page * p.num_kv_heads + h) * (p.block_size / kMxGroup) + offset / kMxGroup) *
                        (nb * kMxBytes);
  uint8_t *kg = p.key_pages + group, *vg = p.value_pages + group;
  constexpr int kAhead = NB > 0 ? NB : 1;  // blocks loaded before any is used
  for (int b0 = 0; b0 < nb; b0 += kAhead) {
    float k8[kAhead][8], v8[kAhead][8];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int u = 0; u < 8; ++u) k8[i][u] = v8[i][u] = 0.f;
      if (slot >= 0) {
        load8<T, VEC>(krow + (b0 + i) * kMxBlock, k8[i]);
        load8<T, VEC>(vrow + (b0 + i) * kMxBlock, v8[i]);
      }
    }
    uint64_t ks = 0, vs = 0;  // scale bytes of the blocks
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      uint32_t byte;
      const uint32_t kw = encode8(k8[i], byte);
      ks |= static_cast<uint64_t>(byte) << (8 * i);
      const uint32_t vw = encode8(v8[i], byte);
      vs |= static_cast<uint64_t>(byte) << (8 * i);
      if (slot < 0) continue;
      const int at = (b0 + i) * kMxBlockBytes + tok * 16 + j * 4;
      *reinterpret_cast<uint32_t *>(kg + at) = kw;
      *reinterpret_cast<uint32_t *>(vg + at) = vw;
    }
    if (slot < 0 || j > 1) continue;
    uint8_t *to = (j ? vg : kg) + nb * kMxBlockBytes + tok * nb + b0;  // lane 0 writes K's, lane 1 V's
    const uint64_t bytes = j ? vs : ks;
    if constexpr (NB == 4) {
      *reinterpret_cast<uint32_t *>(to) = static_cast<uint32_t>(bytes);
    } else if constexpr (NB == 2) {
      *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(bytes);
    } else {
      *to = static_cast<uint8_t>(bytes);
    }
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

// grid (groups of 16 positions x kv heads, 8 warps to a CTA; sequences).  REDO: rows for the dense prefill, which
// notes the sequences that it cannot do.
template <typename T, int NB, bool REDO>
__global__ void __launch_bounds__(256) mxfp4_gather_kernel(const MxGatherParams p, const FastDiv by_heads,
                                                           const FastDiv by_page) {
  pdl_wait();
  const int seq = blockIdx.y;
  const int64_t base = p.cu_seqlens_k[seq];
  const int64_t ctx = p.cu_seqlens_k[seq + 1] - base;
  const int lane = threadIdx.x & 31, j = lane & 3;
  const uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t g = by_heads.div(task);
  const int h = static_cast<int>(task - g * p.num_kv_heads);
  const int64_t pos0 = static_cast<int64_t>(g) * kMxGroup;
  if (pos0 >= ctx || (p.fill && g >= p.fill)) return;
  bool apart = false;  // REDO: this lane's blocks that are not for the dense kernel
  auto note = [&] {    // before the warp returns
    if constexpr (REDO) {
      const bool any = __any_sync(0xffffffffu, apart);
      if (lane == 0) p.redo[(static_cast<int64_t>(seq) * p.num_kv_heads + h) * p.redo_stride + g] = any;
    }
  };
  const int nb = blocks_of<NB>(p.head_dim);
  auto zero_group = [&](int64_t from) {
    for (int tok = lane >> 2; tok < kMxGroup && from + tok < ctx; tok += 8) {
      const int64_t row = base + from + tok;
      if (row < 0 || row >= p.out_rows) continue;
      const int64_t dst = (row * p.num_kv_heads + h) * p.head_dim + j * 8;
      const float zeros[8] = {};
      for (int b = 0; b < nb; ++b) {
        write8(static_cast<T *>(p.out_keys) + dst + b * kMxBlock, zeros);
        write8(static_cast<T *>(p.out_values) + dst + b * kMxBlock, zeros);
      }
    }
  };
  if (p.fill && ctx > static_cast<int64_t>(p.fill) * kMxGroup) {
    if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    apart = true;
    for (int64_t more = g + static_cast<int64_t>(p.fill); more * kMxGroup < min(ctx, p.out_rows); more += p.fill)
      zero_group(more * kMxGroup);
  }
  const int64_t col = by_page.div(g);  // groups of a page
  const int per_page = p.block_size / kMxGroup;
  const int64_t blk = col < p.block_table_stride ? p.block_tables[seq * p.block_table_stride + col] : -1;
  if (blk < 0 || blk >= p.num_blocks) {
    if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    apart = true;  // to be left out, as prefill from the pages does
    if (p.fill) zero_group(pos0);
    note();
    return;
  }
  const int64_t off = ((blk * p.num_kv_heads + h) * per_page + (g - col * per_page)) * (nb * kMxBytes);
  const uint8_t *kg = p.key_pages + off, *vg = p.value_pages + off;
  constexpr int kAhead = NB > 0 ? NB : 1;
  for (int b0 = 0; b0 < nb; b0 += kAhead) {
    uint32_t kw[2][kAhead], vw[2][kAhead];
    uint32_t ks[2][kAhead], vs[2][kAhead];
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // every code and scale is in the page: read whether wanted or not
      const int tok = half * 8 + (lane >> 2);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int code = (b0 + i) * kMxBlockBytes + tok * 16 + j * 4, scale = nb * kMxBlockBytes + tok * nb + b0 + i;
        kw[half][i] = __ldg(reinterpret_cast<const uint32_t *>(kg + code));
        vw[half][i] = __ldg(reinterpret_cast<const uint32_t *>(vg + code));
        ks[half][i] = __ldg(kg + scale);
        vs[half][i] = __ldg(vg + scale);
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int tok = half * 8 + (lane >> 2);
      const int64_t row = base + pos0 + tok;
      if (pos0 + tok >= ctx) continue;
      if constexpr (REDO)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) apart |= mx_apart<T>(false, ks[half][i]) || mx_apart<T>(true, vs[half][i]);
      if (row < 0 || row >= p.out_rows) {
        flag_status(p.status, MI_DEV_BAD_SLOT);
        continue;
      }
      const int64_t dst = (row * p.num_kv_heads + h) * p.head_dim + b0 * kMxBlock + j * 8;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float x[8];
        mx_codes_to_f32(kw[half][i], mx_scale(ks[half][i]), x);
        write8(static_cast<T *>(p.out_keys) + dst + i * kMxBlock, x);
        mx_codes_to_f32(vw[half][i], mx_scale(vs[half][i]), x);
        write8(static_cast<T *>(p.out_values) + dst + i * kMxBlock, x);
      }
    }
  }
  note();
  pdl_launch_dependents();
}

template <typename T, typename I, int NB>
cudaError_t launch_store_tin(const MxStoreParams &p, bool vec, cudaStream_t stream) {
  const int64_t tasks = (p.num_tokens + 7) / 8 * p.num_kv_heads;
  if (tasks >= (int64_t{1} << 31)) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((tasks + 3) / 4)), block(128);
  const FastDiv by_heads(p.num_kv_heads), by_block(p.block_size);
  if (p.num_slots >= (int64_t{1} << 31))
    return vec ? launch_pdl(mxfp4_store_kernel<T, I, true, NB, true>, grid, block, 0, stream, p, by_heads, by_block)
               : launch_pdl(mxfp4_store_kernel<T, I, false, NB, true>, grid, block, 0, stream, p, by_heads, by_block);
  return vec ? launch_pdl(mxfp4_store_kernel<T, I, true, NB, false>, grid, block, 0, stream, p, by_heads, by_block)
             : launch_pdl(mxfp4_store_kernel<T, I, false, NB, false>, grid, block, 0, stream, p, by_heads, by_block);
}

template <typename T, typename I>
cudaError_t launch_store_ti(const MxStoreParams &p, bool vec, cudaStream_t stream) {
  if (p.head_dim == 128) return launch_store_tin<T, I, 4>(p, vec, stream);
  if (p.head_dim == 64) return launch_store_tin<T, I, 2>(p, vec, stream);
  return launch_store_tin<T, I, 0>(p, vec, stream);
}

template <typename T, bool REDO>
cudaError_t launch_gather_t(const MxGatherParams &p, int64_t num_seqs, int64_t max_context, cudaStream_t stream) {
  const int64_t tasks = (max_context + kMxGroup - 1) / kMxGroup * p.num_kv_heads;
  if (tasks >= (int64_t{1} << 31)) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((tasks + 7) / 8), static_cast<unsigned>(num_seqs)), block(256);
  const FastDiv by_heads(p.num_kv_heads), by_page(p.block_size / kMxGroup);
  if (p.head_dim == 128)
    return launch_pdl(mxfp4_gather_kernel<T, 4, REDO>, grid, block, 0, stream, p, by_heads, by_page);
  if constexpr (REDO) return cudaErrorInvalidValue;  // the dense kernel has one head_dim
  if (p.head_dim == 64) return launch_pdl(mxfp4_gather_kernel<T, 2, false>, grid, block, 0, stream, p, by_heads, by_page);
  return launch_pdl(mxfp4_gather_kernel<T, 0, false>, grid, block, 0, stream, p, by_heads, by_page);
}

template <typename T>
cudaError_t launch_store_t(const MxStoreParams &p, int index_dtype, bool vec, cudaStream_t stream) {
  return index_dtype == MI_INDEX_INT32 ? launch_store_ti<T, int32_t>(p, vec, stream)
                                       : launch_store_ti<T, int64_t>(p, vec, stream);
}

}  // namespace

cudaError_t launch_mxfp4_store(const MxStoreParams &p, int dtype, int index_dtype, bool vec,
                               cudaStream_t stream) {
  if (dtype == MI_DTYPE_BFLOAT16) return launch_store_t<__nv_bfloat16>(p, index_dtype, vec, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_store_t<__half>(p, index_dtype, vec, stream);
  return launch_store_t<float>(p, index_dtype, vec, stream);
}

cudaError_t launch_mxfp4_gather(const MxGatherParams &p, int dtype, int64_t num_seqs, int64_t max_context,
                                cudaStream_t stream) {
  if (p.redo != nullptr)
    return dtype == MI_DTYPE_BFLOAT16 ? launch_gather_t<__nv_bfloat16, true>(p, num_seqs, max_context, stream)
                                      : launch_gather_t<__half, true>(p, num_seqs, max_context, stream);
  if (dtype == MI_DTYPE_BFLOAT16) return launch_gather_t<__nv_bfloat16, false>(p, num_seqs, max_context, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_gather_t<__half, false>(p, num_seqs, max_context, stream);
  return launch_gather_t<float, false>(p, num_seqs, max_context, stream);
}

}  // namespace mi
