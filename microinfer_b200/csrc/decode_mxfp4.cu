// Paged decode over the 4-bit cache (layout: mxfp4.cuh): one query token per
// sequence, out = softmax(scale * K q) V with GQA, K and V decoded on the fly.
//
// SIMT form, for every type, head_dim (a multiple of 32 up to 256) and group:
// a CTA of 8 warps takes one (split, kv head x tile of query heads, sequence); a
// warp takes every (8 * splits)-th group of 16 keys.
//   scores: lane (key l / 4, part l % 4) decodes 8 elements of each block of
//           its key and dots them with q (fp32, in shared memory); two shuffles
//           join the four parts;
//   values: lane l owns element l of every block, the accumulators of all
//           heads of the tile in registers, p broadcast from shared memory.
// Online softmax in the log2 domain, everything in fp32.  The splits' states
// (m, l, acc) meet in the workspace and a second launch joins them, so nothing has to
// be zeroed beforehand and no result depends on the order of arrival.
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "params.cuh"

namespace mi {

bool mxfp4_mma_supported(int dtype, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_blocks,
                         int block_size, int64_t capacity);
size_t mxfp4_mma_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t capacity,
                           int sms);
cudaError_t launch_mxfp4_mma(const MxDecodeParams &p, int dtype, cudaStream_t stream);

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kSimtWarps = 8;

// Context of a sequence, clamped to what its block-table row can hold.
__device__ __forceinline__ int mx_context(const MxDecodeParams &p, int64_t seq, bool flag) {
  const int ctx = __ldg(p.context_lens + seq);
  const int64_t cap = p.bt_stride * p.block_size;
  if (ctx <= cap) return ctx > 0 ? ctx : 0;
  if (flag) flag_status(p.status, MI_DEV_BAD_BLOCK);
  return static_cast<int>(cap);
}

template <typename T, int HT, int NB>
__global__ void __launch_bounds__(kSimtWarps * 32) mxfp4_decode_simt_kernel(const MxDecodeParams p) {
  __shared__ float qs[HT][NB * 32];
  __shared__ float ps[kSimtWarps][HT][kMxGroup];
  __shared__ float ml[kSimtWarps][HT][2];
  __shared__ float accs[HT][NB * 32];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, nsplit = gridDim.x;
  const int64_t seq = blockIdx.z;
  const int G = p.num_q_heads / p.num_kv_heads, tiles = (G + HT - 1) / HT;
  const int kvh = blockIdx.y / tiles, h0 = kvh * G + blockIdx.y % tiles * HT;
  const int heads = min(HT, (kvh + 1) * G - h0);
  const int D = p.head_dim, nb = D / kMxBlock;
  const T *query = static_cast<const T *>(p.query) + (seq * p.num_q_heads + h0) * D;
  for (int i = threadIdx.x; i < HT * NB * 32; i += blockDim.x) {
    const int h = i / (NB * 32), d = i % (NB * 32);
    qs[h][d] = h < heads && d < D ? Elem<T>::to_float(query[h * D + d]) * p.scale_log2 : 0.f;
    accs[h][d] = 0.f;
  }
  __syncthreads();

  const int ctx = mx_context(p, seq, threadIdx.x == 0 && split == 0 && blockIdx.y == 0);
  const int groups = (ctx + kMxGroup - 1) / kMxGroup;
  const int32_t *table = p.block_tables + seq * p.bt_stride;
  float m[HT], l[HT], acc[HT][NB];
#pragma unroll
  for (int h = 0; h < HT; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[h][b] = 0.f;
  }
  const int j = lane & 3;
  for (int g = split * kSimtWarps + warp; g < groups; g += nsplit * kSimtWarps) {
    const int pos0 = g * kMxGroup, valid = min(kMxGroup, ctx - pos0);
    const int32_t blk = __ldg(table + pos0 / p.block_size);
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) flag_status(p.status, MI_DEV_BAD_BLOCK);
      continue;
    }
    const int64_t off = mx_group_offset(static_cast<int64_t>(blk) * p.block_size + pos0 % p.block_size, kvh,
                                        p.block_size, p.num_kv_heads, D);
    const uint8_t *kg = p.key_pages + off, *vg = p.value_pages + off;
    float s[HT][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int tok = half * 8 + (lane >> 2);
#pragma unroll
      for (int h = 0; h < HT; ++h) s[h][half] = 0.f;
      for (int b = 0; b < nb; ++b) {
        float k8[8];
        mx_codes_to_f32(*reinterpret_cast<const uint32_t *>(kg + b * kMxBlockBytes + tok * 16 + j * 4),
                        mx_scale(kg[nb * kMxBlockBytes + tok * nb + b]), k8);
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[h][half] = fmaf(k8[i], qs[h][b * 32 + j * 8 + i], s[h][half]);
      }
    }
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      float x[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float t = s[h][half];
        t += __shfl_xor_sync(kAll, t, 1);
        t += __shfl_xor_sync(kAll, t, 2);
        x[half] = half * 8 + (lane >> 2) < valid ? t : -INFINITY;
      }
      float mx = fmaxf(x[0], x[1]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
      const float mn = fmaxf(m[h], mx);
      const float f = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - mn);
      m[h] = mn;
      l[h] *= f;
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[h][b] *= f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tok = half * 8 + (lane >> 2);
        const float pr = tok < valid ? fast_exp2(x[half] - mn) : 0.f;
        if (j == 0) {
          ps[warp][h][tok] = pr;
          l[h] += pr;
        }
      }
    }
    __syncwarp();
    for (int k = 0; k < valid; ++k) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (b >= nb) break;
        const uint32_t byte = vg[b * kMxBlockBytes + k * 16 + lane / 2];
        float v8[8];
        mx_codes_to_f32(lane & 1 ? byte >> 4 : byte & 15u, mx_scale(vg[nb * kMxBlockBytes + k * nb + b]), v8);
#pragma unroll
        for (int h = 0; h < HT; ++h) acc[h][b] = fmaf(ps[warp][h][k], v8[0], acc[h][b]);
      }
    }
    __syncwarp();
  }

  // join the warps
#pragma unroll
  for (int h = 0; h < HT; ++h) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) l[h] += __shfl_xor_sync(kAll, l[h], o);
    if (lane == 0) ml[warp][h][0] = m[h], ml[warp][h][1] = l[h];
  }
  __syncthreads();
  float M[HT], L[HT];
#pragma unroll
  for (int h = 0; h < HT; ++h) {
    M[h] = -INFINITY, L[h] = 0.f;
#pragma unroll
    for (int w = 0; w < kSimtWarps; ++w) M[h] = fmaxf(M[h], ml[w][h][0]);
#pragma unroll
    for (int w = 0; w < kSimtWarps; ++w)
      L[h] += ml[w][h][1] * (ml[w][h][0] == -INFINITY && ml[w][h][1] == 0.f ? 0.f : fast_exp2(ml[w][h][0] - M[h]));
  }
  for (int w = 0; w < kSimtWarps; ++w) {
    if (w == warp) {
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        if (m[h] == -INFINITY && l[h] == 0.f) continue;  // this warp saw no key
        const float f = fast_exp2(m[h] - M[h]);
#pragma unroll
        for (int b = 0; b < NB; ++b) accs[h][b * 32 + lane] += f * acc[h][b];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < HT; ++h) {
    if (h >= heads) break;
    const int64_t row = seq * p.num_q_heads + h0 + h;
    if (nsplit == 1) {
      for (int d = threadIdx.x; d < D; d += blockDim.x)
        static_cast<T *>(p.out)[row * D + d] = Elem<T>::from_float(L[h] == 0.f ? 0.f : accs[h][d] / L[h]);
    } else {
      float *st = p.workspace + (row * nsplit + split) * (D + 2);
      for (int d = threadIdx.x; d < D; d += blockDim.x) st[2 + d] = accs[h][d];
      if (threadIdx.x == 0) st[0] = M[h], st[1] = L[h];
    }
  }
  pdl_launch_dependents();
}

// Join the splits' states: one CTA per (query head, sequence).
template <typename T>
__global__ void __launch_bounds__(128) mxfp4_decode_join_kernel(const MxDecodeParams p, int nsplit) {
  pdl_wait();
  const int D = p.head_dim;
  const int64_t row = static_cast<int64_t>(blockIdx.y) * p.num_q_heads + blockIdx.x;
  const float *st = p.workspace + row * nsplit * (D + 2);
  float M = -INFINITY, L = 0.f;
  for (int s = 0; s < nsplit; ++s) M = fmaxf(M, st[static_cast<int64_t>(s) * (D + 2)]);
  for (int s = 0; s < nsplit; ++s) {
    const float *t = st + static_cast<int64_t>(s) * (D + 2);
    if (t[0] != -INFINITY || t[1] != 0.f) L += t[1] * fast_exp2(t[0] - M);
  }
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float a = 0.f;
    for (int s = 0; s < nsplit; ++s) {
      const float *t = st + static_cast<int64_t>(s) * (D + 2);
      if (t[0] != -INFINITY || t[1] != 0.f) a += t[2 + d] * fast_exp2(t[0] - M);
    }
    static_cast<T *>(p.out)[row * D + d] = Elem<T>::from_float(L == 0.f ? 0.f : a / L);
  }
  pdl_launch_dependents();
}

template <typename T, int HT, int NB>
cudaError_t launch_simt(const MxDecodeParams &p, int nsplit, cudaStream_t stream) {
  const int tiles = (p.num_q_heads / p.num_kv_heads + HT - 1) / HT;
  const dim3 grid(nsplit, p.num_kv_heads * tiles, static_cast<unsigned>(p.num_seqs));
  cudaError_t e = launch_pdl(mxfp4_decode_simt_kernel<T, HT, NB>, grid, dim3(kSimtWarps * 32), 0, stream, p);
  if (e == cudaSuccess && nsplit > 1)
    e = launch_pdl(mxfp4_decode_join_kernel<T>, dim3(p.num_q_heads, static_cast<unsigned>(p.num_seqs)), dim3(128),
                   0, stream, p, nsplit);
  return e;
}

int simt_tile(int G) { return G <= 2 ? 2 : 8; }

template <typename T>
cudaError_t launch_simt_t(const MxDecodeParams &p, int nsplit, cudaStream_t stream) {
  const bool small = simt_tile(p.num_q_heads / p.num_kv_heads) == 2;
  if (p.head_dim <= 128)
    return small ? launch_simt<T, 2, 4>(p, nsplit, stream) : launch_simt<T, 8, 4>(p, nsplit, stream);
  return small ? launch_simt<T, 2, 8>(p, nsplit, stream) : launch_simt<T, 8, 8>(p, nsplit, stream);
}

// Enough CTAs to fill every SM twice, each split at least one group per warp.
int simt_splits(int64_t num_seqs, int num_q_heads, int num_kv_heads, int64_t capacity, int sms) {
  const int G = num_q_heads / num_kv_heads, ht = simt_tile(G);
  const int64_t ctas = num_seqs * num_kv_heads * ((G + ht - 1) / ht);
  int64_t s = 2 * sms / ctas;
  const int64_t most = (capacity + kMxGroup * kSimtWarps - 1) / (kMxGroup * kSimtWarps);
  if (s > most) s = most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}

}  // namespace

size_t mxfp4_decode_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                              int64_t num_blocks, int block_size, int64_t capacity, int sms) {
  if (mxfp4_mma_supported(dtype, num_q_heads, num_kv_heads, head_dim, num_blocks, block_size, capacity))
    return mxfp4_mma_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, capacity, sms);
  const int s = simt_splits(num_seqs, num_q_heads, num_kv_heads, capacity, sms);
  return s == 1 ? 0 : static_cast<size_t>(num_seqs) * num_q_heads * s * (head_dim + 2) * sizeof(float);
}

cudaError_t launch_mxfp4_decode(const MxDecodeParams &p, int dtype, cudaStream_t stream) {
  const int64_t capacity = p.bt_stride * p.block_size;
  if (mxfp4_mma_supported(dtype, p.num_q_heads, p.num_kv_heads, p.head_dim, p.num_blocks, p.block_size, capacity))
    return launch_mxfp4_mma(p, dtype, stream);
  const int s = simt_splits(p.num_seqs, p.num_q_heads, p.num_kv_heads, capacity, sm_count_current());
  if (dtype == MI_DTYPE_BFLOAT16) return launch_simt_t<__nv_bfloat16>(p, s, stream);
  if (dtype == MI_DTYPE_FLOAT16) return launch_simt_t<__half>(p, s, stream);
  return launch_simt_t<float>(p, s, stream);
}

}  // namespace mi
