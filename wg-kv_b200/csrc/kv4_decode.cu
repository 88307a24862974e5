// Ragged paged decode attention over a 4-bit KV cache (format: kv4.cuh).
#include "kv4.cuh"
#include "runtime.h"

namespace wgkv {
namespace {

constexpr int kThreads = 128;
constexpr int kTile = 64;    // tokens per tile
constexpr int kMaxG = 16;

struct Kv4DecodeParams {
  Kv4Pages c;
  const uint16_t* q;
  uint16_t* out;
  const int32_t* seqlens;
  int G;
  float scale_log2;
};

// One CTA per (batch, kv head): tiles of 64 tokens are expanded to fp32 in shared memory, scores by
// dot products, one running maximum and sum per query head; a thread owns one output dimension of every
// query head.
template <int D, int NG>
__global__ void __launch_bounds__(kThreads) kv4_decode_kernel(Kv4DecodeParams p) {
  extern __shared__ float sm[];
  float* ks = sm;                     // [kTile][D + 1]
  float* vs = ks + kTile * (D + 1);   // [kTile][D]
  float* qs = vs + kTile * D;         // [G][D]
  float* ps = qs + kMaxG * D;         // [G][kTile]
  float* ms = ps + kMaxG * kTile;     // [G] running maximum, sum, factor
  float* ls = ms + kMaxG;
  float* fs = ls + kMaxG;
  const int bh = blockIdx.x, tid = threadIdx.x, G = p.G;
  const int cap = p.c.width * p.c.page;
  int len = max(p.seqlens[bh], 0);
  if (len > cap) {
    if (tid == 0) set_error(p.c.err, WGKV_ERR_HEAD_CAPACITY);
    len = cap;
  }
  for (int e = tid; e < G * D; e += kThreads) qs[e] = bf2f(p.q[size_t(bh) * G * D + e]) * p.scale_log2;
  if (tid < G) {
    ms[tid] = -INFINITY;
    ls[tid] = 0.f;
  }
  float acc[kMaxG];
  for (int g = 0; g < kMaxG; ++g) acc[g] = 0.f;
  for (int t0 = 0; t0 < len; t0 += kTile) {
    const int n = min(kTile, len - t0);
    __syncthreads();
    for (int e = tid; e < kTile * 4; e += kThreads) {
      const int r = e >> 2, t = e & 3;
      uint32_t kw[D / 32] = {}, vw[D / 32] = {}, kp[NG] = {}, vp[NG] = {};
      if (r < n) {
        const uint8_t* rec = kv4_record<D, NG>(p.c, bh, t0 + r);
        if (rec) {
          kv4_load_k<D, NG>(rec, (t0 + r) & 15, t, kw, kp);
          kv4_load_v<D, NG>(rec, (t0 + r) & 15, t, vw, vp);
        }
      }
      for (int j = 0; j < D / 32; ++j)
        for (int i = 0; i < 8; ++i) {
          ks[r * (D + 1) + 32 * j + 8 * t + i] = kv4_value((kw[j] >> (4 * i)) & 15u, kp[j * NG / (D / 32)]);
          vs[r * D + 32 * j + 8 * t + i] = kv4_value((vw[j] >> (4 * i)) & 15u, vp[j * NG / (D / 32)]);
        }
    }
    __syncthreads();
    for (int e = tid; e < G * n; e += kThreads) {
      const int g = e / n, r = e - g * n;
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(qs[g * D + d], ks[r * (D + 1) + d], s);
      ps[g * kTile + r] = s;
    }
    __syncthreads();
    if (tid < G) {
      float m = ms[tid];
      for (int r = 0; r < n; ++r) m = fmaxf(m, ps[tid * kTile + r]);
      const float f = exp2f(ms[tid] - m);
      float l = ls[tid] * f;
      for (int r = 0; r < n; ++r) {
        const float x = exp2f(ps[tid * kTile + r] - m);
        ps[tid * kTile + r] = x;
        l += x;
      }
      ms[tid] = m;
      ls[tid] = l;
      fs[tid] = f;
    }
    __syncthreads();
    if (tid < D) {
      for (int g = 0; g < G; ++g) {
        float a = acc[g] * fs[g];
        for (int r = 0; r < n; ++r) a = fmaf(ps[g * kTile + r], vs[r * D + tid], a);
        acc[g] = a;
      }
    }
  }
  __syncthreads();
  if (tid < D)
    for (int g = 0; g < G; ++g)
      p.out[(size_t(bh) * G + g) * D + tid] = f2bf(len > 0 ? acc[g] / ls[g] : 0.f);
}

struct DecodeLaunch {
  Kv4DecodeParams p;
  int BH;
  cudaStream_t stream;
  int status;
  template <int D, int NG>
  void run() {
    const size_t smem = (size_t(kTile) * (2 * D + 1) + kMaxG * D + kMaxG * kTile + 3 * kMaxG) * 4;
    if (cudaFuncSetAttribute(kv4_decode_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) !=
        cudaSuccess) {
      status = WGKV_ECUDA;
      return;
    }
    kv4_decode_kernel<D, NG><<<BH, kThreads, smem, stream>>>(p);
    status = cudaGetLastError() == cudaSuccess ? WGKV_OK : WGKV_ECUDA;
  }
};

}  // namespace
}  // namespace wgkv

using namespace wgkv;

extern "C" size_t wgkv_paged_decode_kv4_workspace_size(int batch, int num_q_heads, int num_kv_heads, int head_dim) {
  return wgkv_paged_decode_workspace_size(batch, num_q_heads, num_kv_heads, head_dim);
}

extern "C" int wgkv_paged_decode_kv4(const uint16_t* q, const uint8_t* cache, int64_t num_pages, int page_size,
                                     int group, const int32_t* cache_seqlens, const int32_t* block_table,
                                     int64_t table_stride, int table_width, int batch, int num_q_heads,
                                     int num_kv_heads, int head_dim, float softmax_scale, uint16_t* out,
                                     void* workspace, size_t workspace_bytes, int* err, void* stream) {
  if (!q || !cache || !cache_seqlens || !block_table || !out || !workspace || !kv4_supported(head_dim, group))
    return WGKV_EINVAL;
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > kMaxG || int64_t(batch) * num_kv_heads > 4096)
    return WGKV_EINVAL;
  if (num_pages <= 0 || page_size <= 0 || page_size % 16 || table_width <= 0 || table_stride < table_width ||
      int64_t(batch) * num_kv_heads * table_width * (page_size / 16) >= (int64_t(1) << 31) ||
      int64_t(table_width) * page_size >= (int64_t(1) << 31) ||
      (reinterpret_cast<uintptr_t>(cache) & 15) || (reinterpret_cast<uintptr_t>(q) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 15))
    return WGKV_EINVAL;
  if (workspace_bytes < wgkv_paged_decode_kv4_workspace_size(batch, num_q_heads, num_kv_heads, head_dim))
    return WGKV_ENOSPC;
  DecodeLaunch a{{{const_cast<uint8_t*>(cache), num_pages, page_size, block_table, table_stride, table_width, err},
                  q, out, cache_seqlens, num_q_heads / num_kv_heads, softmax_scale * 1.4426950408889634f},
                 batch * num_kv_heads, as_stream(stream), WGKV_OK};
  kv4_dispatch(head_dim, group, a);
  return a.status;
}
