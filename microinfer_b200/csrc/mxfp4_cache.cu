// Moving K and V into and out of the 4-bit paged cache (layout: mxfp4.cuh).
//
// Store: for each block of 32 elements x with a = max |x|, the scale is
//   2^e, e = floor(log2 a) - 2  (so that a / 2^e lies in [4, 8), the top binade of e2m1),
// held as the byte e + 127, at least 1; codes are x / 2^e rounded to the
// nearest e2m1 value (ties to even, saturating at 6).  The division by a power
// of two is exact, so codes and scales do not depend on the order of any sum.
// A zero block has the byte 0, a block with an infinity or a NaN the byte 255.
// Four lanes hold a block (8 elements each, one 16-byte load of a 16-bit
// type), two shuffles give a.  Reads 2 or 4 bytes per element and writes 4.25 bits:
// HBM-bound on the read.
//
// Gather: rows of each request in logical order, request-major, as
// code * scale in the requested type (exact in fp32 and bf16 short of
// overflow; fp16 rounds).  One warp per group of 16 tokens and kv head; a lane
// reads 4 bytes of codes (8 elements, 128 consecutive bytes per warp load) and writes
// them as one or two 16-byte vectors.  HBM-bound on the rows that it writes.
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

// Quantise 8 of a block's 32 elements (the quad's lanes hold the rest) and
// write their codes; lane 0 of the quad writes the scale.
__device__ __forceinline__ void store8(const float (&x)[8], uint32_t quad, int j, uint8_t *codes,
                                       uint8_t *scale) {
  uint32_t top = 0;  // largest magnitude as bits: orders like the floats, NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(quad, top, 1));
  top = max(top, __shfl_xor_sync(quad, top, 2));
  uint32_t byte = top >> 23;
  byte = byte > 3 ? byte - 2 : 1;  // the lowest scale is 2^-126
  const float inv = __uint_as_float((254u - byte) << 23);
  uint32_t w = mx_encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv) & 0xffffu;
  w |= mx_encode4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv) << 16;
  if (top == 0) byte = 0;
  if (top >= 0x7f800000u) byte = 255, w = 0;
  *reinterpret_cast<uint32_t *>(codes + j * 4) = w;
  if (j == 0) *scale = static_cast<uint8_t>(byte);
}

// block (bx, by): x walks the row's 8-element vectors, y the tokens.
template <typename T, typename I, bool VEC>
__global__ void __launch_bounds__(256) mxfp4_store_kernel(const MxStoreParams p) {
  pdl_wait();
  const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
  const uint32_t quad = 0xfu << (lane & ~3);
  const int per_head = p.head_dim / 8;
  const int vecs = p.num_kv_heads * per_head;
  const int nb = p.head_dim / kMxBlock;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < p.num_tokens;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int64_t slot = static_cast<int64_t>(static_cast<const I *>(p.slots)[t]);
    if (slot < 0 || slot >= p.num_slots) {
      if (slot != -1 && threadIdx.x == 0) flag_status(p.status, MI_DEV_BAD_SLOT);
      continue;  // every lane of a quad holds the same token
    }
    const T *krow = static_cast<const T *>(p.keys) + t * p.key_stride;
    const T *vrow = static_cast<const T *>(p.values) + t * p.value_stride;
    const int tok = static_cast<int>(slot % kMxGroup);  // block_size is a multiple of the group
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
      float k8[8], v8[8];
      load8<T, VEC>(krow + v * 8, k8);
      load8<T, VEC>(vrow + v * 8, v8);
      const int h = v / per_head, in_head = v - h * per_head;
      const int b = in_head >> 2, j = in_head & 3;
      const int64_t group = mx_group_offset(slot, h, p.block_size, p.num_kv_heads, p.head_dim);
      const int code = b * kMxBlockBytes + tok * 16, scale = nb * kMxBlockBytes + tok * nb + b;
      store8(k8, quad, j, p.key_pages + group + code, p.key_pages + group + scale);
      store8(v8, quad, j, p.value_pages + group + code, p.value_pages + group + scale);
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

// grid (groups of 16 positions x kv heads, 8 warps to a CTA; sequences).
template <typename T>
__global__ void __launch_bounds__(256) mxfp4_gather_kernel(const MxGatherParams p) {
  pdl_wait();
  const int64_t seq = blockIdx.y;
  const int64_t base = p.cu_seqlens_k[seq];
  const int64_t ctx = p.cu_seqlens_k[seq + 1] - base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  const int64_t g = unit / p.num_kv_heads;
  const int h = static_cast<int>(unit - g * p.num_kv_heads);
  const int64_t pos0 = g * kMxGroup;
  if (pos0 < ctx) {
    const int64_t col = pos0 / p.block_size;
    const int64_t blk = col < p.block_table_stride ? p.block_tables[seq * p.block_table_stride + col] : -1;
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
    } else {
      const int nb = p.head_dim / kMxBlock;
      const int64_t off =
          mx_group_offset(blk * p.block_size + pos0 % p.block_size, h, p.block_size, p.num_kv_heads, p.head_dim);
      const int j = lane & 3;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tok = half * 8 + (lane >> 2);
        const int64_t row = base + pos0 + tok;
        if (pos0 + tok >= ctx) continue;
        if (row < 0 || row >= p.out_rows) {
          flag_status(p.status, MI_DEV_BAD_SLOT);
          continue;
        }
        for (int b = 0; b < nb; ++b) {
          const int code = b * kMxBlockBytes + tok * 16 + j * 4, scale = nb * kMxBlockBytes + tok * nb + b;
          const uint32_t kw = *reinterpret_cast<const uint32_t *>(p.key_pages + off + code);
          const uint32_t vw = *reinterpret_cast<const uint32_t *>(p.value_pages + off + code);
          const float ks = mx_scale(p.key_pages[off + scale]), vs = mx_scale(p.value_pages[off + scale]);
          const int64_t dst = (row * p.num_kv_heads + h) * p.head_dim + b * kMxBlock + j * 8;
          float x[8];
          mx_codes_to_f32(kw, ks, x);
          write8(static_cast<T *>(p.out_keys) + dst, x);
          mx_codes_to_f32(vw, vs, x);
          write8(static_cast<T *>(p.out_values) + dst, x);
        }
      }
    }
  }
  pdl_launch_dependents();
}

template <typename T, typename I>
cudaError_t launch_store_ti(const MxStoreParams &p, bool vec, cudaStream_t stream) {
  const int vecs = p.num_kv_heads * (p.head_dim / 8);
  const int bx = vecs < 256 ? vecs : 256, by = 256 / bx;
  int64_t blocks = (p.num_tokens + by - 1) / by;
  const int64_t cap = static_cast<int64_t>(sm_count_current()) * 16;
  if (blocks > cap) blocks = cap;
  const dim3 grid(static_cast<unsigned>(blocks)), block(bx, by);
  return vec ? launch_pdl(mxfp4_store_kernel<T, I, true>, grid, block, 0, stream, p)
             : launch_pdl(mxfp4_store_kernel<T, I, false>, grid, block, 0, stream, p);
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
  const int64_t units = (max_context + kMxGroup - 1) / kMxGroup * p.num_kv_heads;
  const dim3 grid(static_cast<unsigned>((units + 7) / 8), static_cast<unsigned>(num_seqs));
  if (dtype == MI_DTYPE_BFLOAT16)
    return launch_pdl(mxfp4_gather_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, p);
  if (dtype == MI_DTYPE_FLOAT16)
    return launch_pdl(mxfp4_gather_kernel<__half>, grid, dim3(256), 0, stream, p);
  return launch_pdl(mxfp4_gather_kernel<float>, grid, dim3(256), 0, stream, p);
}

}  // namespace mi
